// ttt_lce.hip — the softmax cross entropy of a linear head for gfx950:
// forward, backward, double backward (formulas in include/ttt_ops.h), and
// their C entry points.
//
// Everything is tile products (ttt_gemm.h) with work done on the tiles where
// they are made:
//   forward    z tiles -> per tile and token (max, sum of exponentials)
//   backward   z tiles again -> G = c (p - 1_t); then the products dX = G W
//              and dW = G^T X
//   gg         z and U tiles -> H (and G); then [H|G][W;B] and [H^T|G^T][X;A]
// z is formed again instead of kept: 2 N V d operations against 4 N V bytes
// written and read.  G and H exist for one piece of the vocabulary at a time
// (kPieceBytes), so memory does not grow with N V.
//
// H needs h_i = sum_j p_ij U_ij before its tiles.  As U = A W^T + X B^T,
//   h_i = A_i . (sum_j p_ij W_j) + X_i . (sum_j p_ij B_j)
//       = (A_i . dX_i + X_i . (G B)_i) / c_i + U_{i,t_i}
// where dX is the backward's and G B a product that gX has anyway: a dot
// product per row in place of a pass over z and U (4 or 6 N V d operations).
// Only where the upstream gradient's own gradient is asked for (c may be 0
// there), or dX is not given, are the sums formed from tiles.
//
// 16-bit types: G and H are rounded once to the operands' type, scaled by one
// factor for all rows (k_factors) that products undo in fp32.  bf16: c over
// the largest |c|, so that rows which count alike are rounded like p - 1_t
// itself (one c for all would round the targets' entries, near -c, all to the
// same side).  fp16: the same with the largest entry at kF16Scale, since a
// softmax over a large vocabulary is below fp16's smallest values.  What the
// rounding takes from a row's target, its largest entry as a rule, is kept in
// fp32 and comes back, times the target's row of W (or B), where the sums over
// the vocabulary are stored.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/ttt_ops.h"
#include "ttt_gemm.h"
#include "ttt_ops.h"

namespace ttt {
namespace {

constexpr float kF16Scale = 16384.f;  // the largest stored magnitude: room below fp16's 65504 for rounding

__host__ __device__ __forceinline__ int round8(int x) { return (x + 7) & ~7; }
// Row stride of G and H of m columns: whole 128-byte lines of 16-bit values.
__host__ __device__ __forceinline__ int piece_ld(int m) { return (m + 63) / 64 * 64; }

// ---------------------------------------------------------------------------
// Row copies of 16-bit operands: padded to 8 columns (zeros), and zeros in the
// rows that do not count, which meet factors of 0 in a sum over the rows.
// ---------------------------------------------------------------------------
struct CopyArgs {
  const void* src;  // [R, C], row stride ld
  int64_t ld;
  int R, C;
  void* dst;           // [R][round8(C)]
  const float* live;   // or null: rows of 0 are left out
};

__global__ __launch_bounds__(256) void k_copy_rows(CopyArgs a) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);  // a wave a row
  if (row >= a.R) return;
  const uint16_t* s = (const uint16_t*)a.src + row * a.ld;
  const int width = round8(a.C);
  uint16_t* d = (uint16_t*)a.dst + (int64_t)row * width;
  const bool live = !a.live || a.live[row] != 0.f;
  for (int c = 8 * (threadIdx.x & 63); c < width; c += 512) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (live) {
      if (c + 8 <= a.C) {
        __builtin_memcpy(&v, s + c, 16);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j / 2] |= c + j < a.C ? (uint32_t)s[c + j] << (16 * (j & 1)) : 0u;
      }
    }
    *(u32x4*)(d + c) = v;
  }
}

// ---------------------------------------------------------------------------
// The products' tile shapes.  16-bit: 256 x 256 (eight waves of 128 x 64), with
// one accumulator, and 128 x 128 (four of 64 x 64).  fp32: 128 x 128 (eight of
// 64 x 32) and 64 x 128 (four of 32 x 64).  Logits of few tokens or few tiles:
// 32 x 32 (DirectProduct).
// ---------------------------------------------------------------------------
enum : int { kDirect = 0, kSmall = 1, kBig = 2 };

template <typename T, bool MT, bool NT, int SIZE>
struct ProductOf {
  static constexpr bool big = SIZE == kBig;
  typedef TileProduct<T, big ? 256 : 128, big ? 256 : 128, 2, big ? 4 : 2, MT, NT> type;
};
template <bool MT, bool NT, int SIZE>
struct ProductOf<float, MT, NT, SIZE> {
  static constexpr bool big = SIZE == kBig;
  typedef SplitProduct<big ? 128 : 64, 128, 2, big ? 4 : 2, MT, NT> type;
};
template <typename T>
struct ProductOf<T, false, false, kDirect> {
  typedef DirectProduct<T> type;
};
template <>
struct ProductOf<float, false, false, kDirect> {
  typedef DirectProduct<float> type;
};

template <typename T, int SIZE>
constexpr int kThreadsOf = SIZE == kBig ? 512 : 256;

template <typename T, typename P>
__device__ __forceinline__ typename P::Lds lds_of() {
  if constexpr (P::BM > 32) {
    __shared__ __attribute__((aligned(16))) char m0[P::kBytesM], m1[P::kBytesM], n0[P::kBytesN], n1[P::kBytesN];
    return {m0, m1, n0, n1};
  } else {
    __shared__ __attribute__((aligned(16))) char m[P::kBytesM], n[P::kBytesN];
    return {m, n};
  }
}

template <typename T, typename P>
__device__ __forceinline__ P product_at(int m0, int n0, int M, int N, const float* live) {
  if constexpr (sizeof(T) == 2 || P::BM == 32) return P(m0, n0, M, N);
  else return P(m0, n0, M, N, live);
}

// ---------------------------------------------------------------------------
// z tiles and what is made of them.
// ---------------------------------------------------------------------------
enum : int { kStats = 0, kGrad = 1, kHSum = 2, kHGrad = 3 };

struct ZArgs {
  SegList z, u;
  int M, N;  // vocabulary rows of the piece, tokens
  int tm, tn;
  int v0;  // the piece's first vocabulary row
  const int64_t* target;
  const float* stat;  // [N] row max, [N] 1 / sum of exponentials
  float2* part;       // [parts][N]: (max, sum) | (sum p U, -)
  float* at_target;   // [N]: z or U at the target
  const float* h;     // [N]
  const float* q;     // [N]: h - U at the target
  const float* colmul;  // [N]
  float *rest_g, *rest_h;  // [N]: what rounding took from G and H at the target (16-bit)
  void *g, *hh;       // G and H, [N][piece_ld(M)], or null
};

// A wave's tile to the rows of a [N][piece_ld(M)] matrix.  val(i, j): the lane's
// four values of acc[i][j], 0 past M.  16-bit: through the wave's own LDS, so
// that global stores are whole 128-byte rows.
template <typename P, typename T, typename F>
__device__ __forceinline__ void store_tile(const P& tp, char* lds, void* out, int M, int N, F val) {
  constexpr int MI = P::MI, NI = P::NI;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int ld = piece_ld(M);
  T* o = (T*)out;
  if constexpr (sizeof(T) == 4 || MI == 1) {
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int n = tp.n_of(j), m = tp.m_of(i);
        const f32x4 v = val(i, j);
        if (n < N && m < ld) {
          const T q[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
          __builtin_memcpy(o + (int64_t)n * ld + m, q, sizeof(q));
        }
      }
  } else {
    constexpr int RB = MI * 32, CH = RB / 16;  // row bytes, chunks
    typedef T t2 __attribute__((ext_vector_type(2)));
    char* w = lds + 16 * RB * tp.wave;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const f32x4 v = val(i, j);
        const t2 u[2] = {__builtin_convertvector(f32x2{v[0], v[1]}, t2), __builtin_convertvector(f32x2{v[2], v[3]}, t2)};
        __builtin_memcpy(w + c * RB + 16 * ((2 * i + (g >> 1)) ^ (c & 7)) + 8 * (g & 1), u, 8);
      }
#pragma unroll
      for (int t = 0; t < CH / 4; ++t) {
        const int r = t * (64 / CH) + lane / CH, ch = lane % CH;
        const u32x4 u = *(const u32x4*)(w + r * RB + 16 * (ch ^ (r & 7)));
        const int n = tp.n0 + (tp.wn * NI + j) * 16 + r, m = tp.m0 + tp.wm * MI * 16 + 8 * ch;
        if (n < N && m < ld) *(u32x4*)(o + (int64_t)n * ld + m) = u;
      }
    }
  }
}

template <typename T, int MODE, int SIZE>
__global__ __launch_bounds__((kThreadsOf<T, SIZE>), 2) void k_logits(ZArgs a) {
  constexpr bool kDual = MODE >= kHSum;
  typedef typename ProductOf<T, false, false, SIZE>::type P;
  constexpr int MI = P::MI, NI = P::NI;
  const typename P::Lds lds = lds_of<T, P>();
  int tm, tn;
  tile_of(blockIdx.x, a.tm, a.tn, &tm, &tn);
  P tp = product_at<T, P>(tm * P::BM, tn * P::BN, a.M, a.N, nullptr);
  f32x4 z[MI][NI], u[kDual ? MI : 1][kDual ? NI : 1];
  P::zero(z);
  tp.run(z, a.z, 0, list_steps<P::kStep>(a.z), lds);
  if constexpr (kDual) {
    P::zero(u);
    tp.run(u, a.u, 0, list_steps<P::kStep>(a.u), lds);
  }
  // Nothing from here on overlaps the products, so it is kept short: rows past
  // M are made to count for nothing beforehand, where there are any, and the
  // target, which few waves have, is put in afterwards.  In place of a test of
  // both at every value (4096 x 1024 x 16384 bf16): forward 147 -> 132 us,
  // backward 163 -> 146, double backward 344 -> 328.
  if (tp.mrows < P::BM) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (tp.m_of(i) + e >= a.M)
#pragma unroll
          for (int j = 0; j < NI; ++j) z[i][j][e] = -__builtin_inff();
  }
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int n = tp.n_of(j);
    const bool nin = n < a.N;
    const int64_t td = nin ? a.target[n] - a.v0 : -1;  // the target's row in the piece
    // the target is value e of acc[i] for at = 16 i + e
    const int at = td >= 0 && td < a.M ? (int)td - tp.m_of(0) : -1;
    const bool hit = at >= 0 && at < 16 * MI && (at & 12) == 0;
    const auto pick = [&](const auto& acc) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) v = at == 16 * i + e ? acc[i][j][e] : v;
      return v;
    };
    const auto put = [&](auto& acc, float v) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = at == 16 * i + e ? v : acc[i][j][e];
    };
    if constexpr (MODE == kStats) {
      float mx = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, z[i][j][e]);
      mx = group_max(mx);
      const float about = mx == -__builtin_inff() ? 0.f : mx;  // a wave whose rows are all past M: 0
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += fast_exp2((z[i][j][e] - about) * kLog2e);
      s = group_sum(s);
      if (g == 0 && nin) a.part[((int64_t)(tm * P::WM + tp.wm)) * a.N + n] = make_float2(mx, s);
      if (hit) a.at_target[n] = pick(z);
    } else {
      const float mx = nin ? a.stat[n] : 0.f, inv = nin ? a.stat[a.N + n] : 0.f;
      if constexpr (MODE == kHSum) {
        float hs = 0.f;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) hs += fast_exp2((z[i][j][e] - mx) * kLog2e) * u[i][j][e];
        hs = group_sum(hs) * inv;
        if (g == 0 && nin) a.part[((int64_t)(tm * P::WM + tp.wm)) * a.N + n] = make_float2(hs, 0.f);
        if (hit) a.at_target[n] = pick(u);
      } else {
        const float cm = nin ? a.colmul[n] : 0.f, h = MODE == kHGrad && nin ? a.h[n] : 0.f, ci = cm * inv;
        const bool live = cm != 0.f;  // rows that do not count: 0 whatever their logits are
        const float zt = hit ? pick(z) : 0.f;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float cp = fast_exp2((z[i][j][e] - mx) * kLog2e) * ci;
            if constexpr (MODE == kHGrad) u[i][j][e] = live ? cp * (u[i][j][e] - h) : 0.f;
            z[i][j][e] = live ? cp : 0.f;
          }
        if (hit) {
          const float p = fast_exp2((zt - mx) * kLog2e) * inv, gt = live ? cm * (p - 1.f) : 0.f;
          put(z, gt);
          if (sizeof(T) == 2 && a.rest_g) a.rest_g[n] = gt - (float)(T)gt;
          if constexpr (MODE == kHGrad) {
            // from q: U there and h come from different sums, and p near 1 has their difference small
            const float ht = live ? -cm * p * a.q[n] : 0.f;
            put(u, ht);
            if (sizeof(T) == 2 && a.rest_h) a.rest_h[n] = ht - (float)(T)ht;
          }
        }
      }
    }
  }
  if constexpr (MODE == kGrad || MODE == kHGrad) {
    char* at;
    if constexpr (SIZE != kDirect) at = lds.m0;
    else at = lds.m;
    if constexpr (kDual)
      if (a.hh) store_tile<P, T>(tp, at, a.hh, a.M, a.N, [&](int i, int j) { return u[i][j]; });
    if (a.g) store_tile<P, T>(tp, at, a.g, a.M, a.N, [&](int i, int j) { return z[i][j]; });
  }
}

// Rows of W and B at the targets, times what rounding took there.
struct Rest {
  const int64_t* target;
  int V;
  const void *w, *b;  // or null
  int64_t ldw, ldb;
  const float *rw, *rb;
};

template <typename T>
__device__ __forceinline__ float rest_at(const Rest& a, int n, int m) {
  float v = 0.f;
  if constexpr (sizeof(T) == 2) {
    const int64_t t = a.target ? a.target[n] : -1;
    if (t >= 0 && t < a.V) {
      if (a.w) v += a.rw[n] * (float)((const T*)a.w)[t * a.ldw + m];
      if (a.b) v += a.rb[n] * (float)((const T*)a.b)[t * a.ldb + m];
    }
  }
  return v;
}

// ---------------------------------------------------------------------------
// Plain products: out[n][m] = alpha * sum_k, to the output (and its fp32 copy),
// or as fp32 to part[split][N][M] (added to what is there from earlier pieces).
// ---------------------------------------------------------------------------
struct OutArgs {
  SegList l;
  int M, N, tm, tn;
  int split, chunk;  // workgroups per tile, steps of each
  float* part;       // or null: direct
  int add;
  void* out;
  int64_t ld;
  float* out32;       // [N][M] or null
  const float* rows;  // [N] or null: rows that do not count (0) are 0
  const float* live;  // turned fp32 M operand: the k that do not count are left out
  const float* alpha;
  Rest rest;
};

template <typename T, bool NT, int SIZE>
__global__ __launch_bounds__((kThreadsOf<T, SIZE>), 2) void k_product(OutArgs a) {
  typedef typename ProductOf<T, true, NT, SIZE>::type P;
  constexpr int MI = P::MI, NI = P::NI;
  const typename P::Lds lds = lds_of<T, P>();
  const int s = blockIdx.x / (a.tm * a.tn), id = blockIdx.x % (a.tm * a.tn);
  int tm, tn;
  tile_of(id, a.tm, a.tn, &tm, &tn);
  P tp = product_at<T, P>(tm * P::BM, tn * P::BN, a.M, a.N, a.live);
  f32x4 acc[MI][NI];
  P::zero(acc);
  const int steps = list_steps<P::kStep>(a.l), lo = s * a.chunk, hi = lo + a.chunk < steps ? lo + a.chunk : steps;
  tp.run(acc, a.l, lo, hi, lds);
  const float al = a.part ? 1.f : *a.alpha;
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int n = tp.n_of(j);
    if (n >= a.N) continue;
    const bool dead = !a.part && a.rows && a.rows[n] == 0.f;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = tp.m_of(i);
      if (m >= a.M) continue;
      const int cnt = a.M - m < 4 ? a.M - m : 4;
      f32x4 v = acc[i][j];
      if (a.part) {
        float* o = a.part + ((int64_t)s * a.N + n) * a.M + m;
        if (cnt == 4) {
          f32x4 old = {0.f, 0.f, 0.f, 0.f};
          if (a.add) __builtin_memcpy(&old, o, 16);
          v += old;
          __builtin_memcpy(o, &v, 16);
        } else {
          for (int e = 0; e < cnt; ++e) o[e] = a.add ? o[e] + v[e] : v[e];
        }
      } else {
        if constexpr (!NT)
          for (int e = 0; e < cnt; ++e) v[e] += rest_at<T>(a.rest, n, m + e);
        v = dead ? f32x4{0.f, 0.f, 0.f, 0.f} : v * al;
        T* o = (T*)a.out + (int64_t)n * a.ld + m;
        float* o32 = a.out32 ? a.out32 + (int64_t)n * a.M + m : nullptr;
        if (cnt == 4) {
          const T r[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
          __builtin_memcpy(o, r, sizeof(r));
          if (o32) __builtin_memcpy(o32, &v, 16);
        } else {
          for (int e = 0; e < cnt; ++e) {
            o[e] = (T)v[e];
            if (o32) o32[e] = v[e];
          }
        }
      }
    }
  }
}

// out[n][m] = alpha * sum of the splits' parts, in their order.
template <typename T>
__global__ __launch_bounds__(256) void k_finish(OutArgs a) {
  const int64_t total = (int64_t)a.N * a.M, i4 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i4 >= total) return;
  const float al = *a.alpha;
  const int cnt = total - i4 < 4 ? (int)(total - i4) : 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.split; ++s) {
    const float* p = a.part + s * total + i4;
    if (cnt == 4) {
      f32x4 t;
      __builtin_memcpy(&t, p, 16);
      v += t;
    } else {
      for (int e = 0; e < cnt; ++e) v[e] += p[e];
    }
  }
  int n = (int)(i4 / a.M), m = (int)(i4 % a.M);
  if (cnt == 4 && m + 4 <= a.M) {
    for (int e = 0; e < 4; ++e) v[e] += rest_at<T>(a.rest, n, m + e);
    v = a.rows && a.rows[n] == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : v * al;
    const T r[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    __builtin_memcpy((T*)a.out + n * a.ld + m, r, sizeof(r));
    if (a.out32) __builtin_memcpy(a.out32 + i4, &v, 16);
    return;
  }
  for (int e = 0; e < cnt; ++e) {
    const float r = a.rows && a.rows[n] == 0.f ? 0.f : (v[e] + rest_at<T>(a.rest, n, m)) * al;
    ((T*)a.out)[n * a.ld + m] = (T)r;
    if (a.out32) a.out32[i4 + e] = r;
    if (++m == a.M) {
      m = 0;
      ++n;
    }
  }
}

// ---------------------------------------------------------------------------
// Row kernels.
// ---------------------------------------------------------------------------
struct RowArgs {
  int N, V, parts, reduction, dtype;
  int64_t ignore;
  const int64_t* target;
  const float* weight;  // row weights or null
  const float2* part;
  const float* at_target;
  const float* grad_loss;
  float* stat;  // [2N + 2]: max, 1/sum, 1/denominator, weight sum
  float* row;   // [N]: the rows' losses | the rows' shares of the upstream gradient's gradient
  float2* sums;  // [ceil(N / 64)]: sums of losses and weights
  float* out;   // reduced
  float *h, *q;
  float *coef, *live, *colmul, *alpha;
  const float *nx, *na, *nw, *nb;  // row norms of X, A, W, B (fp16 gg), or null
};

__device__ __forceinline__ float row_weight(const RowArgs& a, int n) {
  return a.target[n] == a.ignore ? 0.f : a.weight ? a.weight[n] : 1.f;
}
__device__ __forceinline__ bool bad_target(const RowArgs& a, int n) { return a.target[n] < 0 || a.target[n] >= a.V; }

// (max, sum of exponentials about it) of two sets.
__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
  const float mx = fmaxf(a.x, b.x);
  return make_float2(mx, (a.y == 0.f ? 0.f : a.y * fast_exp2((a.x - mx) * kLog2e)) +
                             (b.y == 0.f ? 0.f : b.y * fast_exp2((b.x - mx) * kLog2e)));
}

template <bool STATS>
__device__ __forceinline__ float2 join_two(float2 a, float2 b) {
  if constexpr (STATS) return join_stats(a, b);
  else return make_float2(a.x + b.x, 0.f);
}

// The parts' results of 64 tokens a workgroup, to the lanes of wave 0: lane l
// has token *n (N: none).  All 1024 threads read parts, for fewer than 33
// tokens too, where a wave takes several parts at once (1 token, 256 parts: 3.9
// us in place of 5.5).
template <bool STATS>
__device__ __forceinline__ float2 join_parts(const float2* part, int parts, int N, int* n, float2 (*lds)[64]) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int lanes = 64;
  while (lanes / 2 >= N) lanes /= 2;  // lanes of a part
  *n = blockIdx.x * 64 + lane % lanes;
  float2 s = make_float2(STATS ? -__builtin_inff() : 0.f, 0.f);
  if (*n < N)
#pragma unroll 4
    for (int i = (int)threadIdx.x / lanes; i < parts; i += 1024 / lanes)
      s = join_two<STATS>(s, part[(int64_t)i * N + *n]);
  for (int m = lanes; m < 64; m <<= 1) s = join_two<STATS>(s, make_float2(__shfl_xor(s.x, m), __shfl_xor(s.y, m)));
  lds[w][lane] = s;
  __syncthreads();
  if (w == 0)
    for (int i = 1; i < 16; ++i) s = join_two<STATS>(s, lds[i][lane]);
  if (lane >= lanes) *n = N;
  return s;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// The sums of the rows' losses and weights to the loss and its denominator.
__device__ __forceinline__ void finish_loss(const RowArgs& a, float l, float w) {
  if (threadIdx.x != 0) return;
  const float inv = a.reduction == TTT_REDUCE_MEAN ? 1.f / fmaxf(w, 1.f) : 1.f;
  a.stat[2 * a.N] = inv;
  a.stat[2 * a.N + 1] = w;
  if (a.reduction != TTT_REDUCE_NONE) a.out[0] = l * inv;
}

// The tiles' (max, sum) to the row's, and its loss: log(sum) - (z_t - max),
// which keeps its digits where the target has nearly all of the probability.
__global__ __launch_bounds__(1024) void k_join_loss(RowArgs a) {
  __shared__ float2 lds[16][64];
  int n;
  const float2 s = join_parts<true>(a.part, a.parts, a.N, &n, lds);
  if (threadIdx.x >= 64) return;
  float w = 0.f, wl = 0.f;
  if (n < a.N) {
    a.stat[n] = s.x;
    a.stat[a.N + n] = 1.f / s.y;
    w = row_weight(a, n);
    const float l = bad_target(a, n) ? __builtin_nanf("") : logf(s.y) - (a.at_target[n] - s.x);
    wl = w == 0.f ? 0.f : w * l;
    a.row[n] = wl;
  }
  wl = wave_sum(wl);
  w = wave_sum(w);
  // one workgroup (or nothing to reduce): the whole reduction is here
  if (gridDim.x == 1 || (a.reduction == TTT_REDUCE_NONE && blockIdx.x == 0)) finish_loss(a, wl, w);
  else if (threadIdx.x == 0) a.sums[blockIdx.x] = make_float2(wl, w);
}

// h = sum p U, and the rows' shares of the upstream gradient's gradient.
__global__ __launch_bounds__(1024) void k_join_h(RowArgs a) {
  __shared__ float2 lds[16][64];
  int n;
  const float2 s = join_parts<false>(a.part, a.parts, a.N, &n, lds);
  if (threadIdx.x >= 64 || n >= a.N) return;
  a.h[n] = s.x;
  a.q[n] = s.x - a.at_target[n];
  if (a.row) {
    const float w = row_weight(a, n);
    a.row[n] = w == 0.f ? 0.f
               : bad_target(a, n) ? __builtin_nanf("")
                                  : w * a.stat[2 * a.N] * (s.x - a.at_target[n]);
  }
}

// Rows 0 .. parts - 1 of the tiles' partial results to row 0, so that what is
// kept does not grow with the vocabulary.
template <bool STATS>
__global__ __launch_bounds__(1024) void k_merge(float2* part, int parts, int N) {
  __shared__ float2 lds[16][64];
  int n;
  const float2 s = join_parts<STATS>(part, parts, N, &n, lds);
  if (threadIdx.x < 64 && n < N) part[n] = s;
}

// A workgroup's sum in a fixed order.
__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) t += lds[i];
  return t;
}
__device__ __forceinline__ float block_max(float v, float* lds) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = fmaxf(v, __shfl_xor(v, m));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = lds[0];
  for (int i = 1; i < (int)(blockDim.x >> 6); ++i) t = fmaxf(t, lds[i]);
  return t;
}

// One workgroup: the sums of the workgroups of k_join_loss to the loss and its denominator.
__global__ __launch_bounds__(1024) void k_reduce_loss(RowArgs a) {
  __shared__ float lds[16];
  float l = 0.f, w = 0.f;
  for (int i = threadIdx.x; i < (a.N + 63) / 64; i += 1024) {
    l += a.sums[i].x;
    w += a.sums[i].y;
  }
  l = block_sum(l, lds);
  w = block_sum(w, lds);
  finish_loss(a, l, w);
}

// The rows' coefficients c, which rows count, and the factors that G and H are stored with:
// colmul, undone by alpha.  One workgroup for 16-bit types: it finds the
// largest |c| (fp16 gg: times a bound of the row's |U - h|, 2 max |U| <= 2
// (|A_i| max |W_j| + |X_i| max |B_j|)) first.
__global__ __launch_bounds__(1024) void k_factors(RowArgs a) {
  __shared__ float lds[16];
  const float inv = a.stat[2 * a.N];
  float wm = 0.f, bm = 0.f, top = 0.f;
  if (a.nw || a.nb) {
    for (int v = threadIdx.x; v < a.V; v += 1024) {
      if (a.nw) wm = fmaxf(wm, a.nw[v]);
      if (a.nb) bm = fmaxf(bm, a.nb[v]);
    }
    wm = block_max(wm, lds);
    bm = block_max(bm, lds);
  }
  // kRows rows of a thread at a time: their loads, then the rest
  constexpr int kRows = 4;
  const int stride = gridDim.x * 1024;
  for (int n0 = blockIdx.x * 1024 + threadIdx.x; n0 < a.N; n0 += kRows * stride) {
    int64_t t[kRows];
    float w[kRows], up[kRows], ub[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int n = n0 + i * stride;
      const bool in = n < a.N;
      t[i] = in ? a.target[n] : a.ignore;
      w[i] = in && a.weight ? a.weight[n] : 1.f;
      up[i] = in ? a.grad_loss[a.reduction == TTT_REDUCE_NONE ? n : 0] : 0.f;
      ub[i] = (in && a.na ? a.na[n] * wm : 0.f) + (in && a.nx ? a.nx[n] * bm : 0.f);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int n = n0 + i * stride;
      if (n >= a.N) break;
      if (t[i] == a.ignore) w[i] = 0.f;
      const float c = w[i] == 0.f ? 0.f : t[i] < 0 || t[i] >= a.V ? __builtin_nanf("") : up[i] * w[i] * inv;
      a.coef[n] = c;
      a.live[n] = w[i] == 0.f ? 0.f : 1.f;
      if (a.dtype == TTT_F32) a.colmul[n] = c;
      const float m = fabsf(c) * (a.nw || a.nb ? fmaxf(1.f, 2.f * ub[i]) : 1.f);
      if (c != 0.f && m < __builtin_inff()) top = fmaxf(top, m);
    }
  }
  if (a.dtype == TTT_F32) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.alpha = 1.f;
    return;
  }
  top = fmaxf(block_max(top, lds), 1e-30f);
  const float s = (a.dtype == TTT_F16 ? kF16Scale : 1.f) / top;
  for (int n0 = threadIdx.x; n0 < a.N; n0 += kRows * 1024) {  // this thread's rows of before
    float c[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) c[i] = n0 + i * 1024 < a.N ? a.coef[n0 + i * 1024] : 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (n0 + i * 1024 < a.N) a.colmul[n0 + i * 1024] = c[i] * s;
  }
  if (threadIdx.x == 0) *a.alpha = a.dtype == TTT_F16 ? top * (1.f / kF16Scale) : top;
}

__global__ __launch_bounds__(1024) void k_sum(const float* x, int n, float* out) {
  __shared__ float lds[16];
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) s += x[i];
  s = block_sum(s, lds);
  if (threadIdx.x == 0) *out = s;
}

// norm[r] = |row r| of up to four operands in one launch, a wave a row.
struct NormList {
  struct {
    const void* x;
    int64_t ld;
    int rows;
    float* norm;
  } s[4];
  int n, cols;
};

template <typename T>
__global__ __launch_bounds__(256) void k_norms(NormList a) {
  int r = blockIdx.x * 4 + (threadIdx.x >> 6), i = 0;
  const int lane = threadIdx.x & 63;
  for (; i < a.n && r >= a.s[i].rows; ++i) r -= a.s[i].rows;
  if (i >= a.n) return;
  const T* x = (const T*)a.s[i].x + r * a.s[i].ld;
  float s = 0.f;
#pragma unroll 4
  for (int c = lane; c < a.cols; c += 64) {
    const float v = (float)x[c];
    s += v * v;
  }
  s = wave_sum(s);
  if (lane == 0) a.s[i].norm[r] = sqrtf(s);
}

struct HArgs {
  int N, V, d, split;
  const int64_t* target;
  const float *coef, *alpha;
  const void *x, *w, *a, *b;  // a, b: or null
  int64_t ldx, ldw, lda, ldb;
  const float* dx32;  // [N][d]: the backward's dX (with a)
  const float* gb;    // [split][N][d]: G B (with b), over alpha
  const float* rest;  // [N]: what rounding took from G at the target, over alpha (16-bit)
  float *h, *q;
};

// q_i = (A_i . dX_i + X_i . (G B)_i) / c_i and h_i = q_i + A_i . W_t + X_i . B_t: a
// wave a row.
template <typename T>
__global__ __launch_bounds__(256) void k_row_h(HArgs a) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= a.N) return;
  const float c = a.coef[n];
  if (!(c != 0.f) || c != c) {  // uniform: a row that does not count, or a target that does not exist
    if (lane == 0) a.h[n] = a.q[n] = 0.f;
    return;
  }
  const int64_t t = a.target[n], n64 = n;
  const float al = *a.alpha;
  float s = 0.f, u = 0.f;
  for (int i = lane; i < a.d; i += 64) {
    if (a.a) {
      const float v = (float)((const T*)a.a)[n64 * a.lda + i];
      s += v * a.dx32[n64 * a.d + i];
      u += v * (float)((const T*)a.w)[t * a.ldw + i];
    }
    if (a.b) {
      const float v = (float)((const T*)a.x)[n64 * a.ldx + i];
      float q = 0.f;
#pragma unroll 4
      for (int k = 0; k < a.split; ++k) q += a.gb[((int64_t)k * a.N + n64) * a.d + i];
      const float bt = (float)((const T*)a.b)[t * a.ldb + i];
      if (sizeof(T) == 2) q += a.rest[n] * bt;
      s += v * (q * al);
      u += v * bt;
    }
  }
  s = wave_sum(s);
  u = wave_sum(u);
  if (lane == 0) {
    a.q[n] = s / c;
    a.h[n] = s / c + u;
  }
}

// ---------------------------------------------------------------------------
// Host: sizes, workspace layout, launches.
// ---------------------------------------------------------------------------
constexpr int64_t kPieceBytes = 512ll << 20;  // G (and H) of a piece
constexpr int64_t kPackBytes = 256ll << 20;   // copied head rows of a piece
constexpr int64_t kPartBytes = 64ll << 20;    // the tiles' partial results that are kept before they are merged
constexpr int kPieceRows = 131072;            // vocabulary rows of a piece at most
constexpr int kMaxSplit = 64;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Plan {
  int dtype, entry, N, V, d, dp, es;
  bool f32, pack;  // pack: 16-bit rows are copied (not a multiple of 8 columns)
  int vc, pieces;  // vocabulary rows of a piece
};

// Hands out 256-byte aligned parts of the workspace; without one, counts.
struct Carver {
  char* base;
  int64_t used;
  void* take(int64_t bytes) {
    void* r = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return r;
  }
  float* floats(int64_t n) { return (float*)take(n * 4); }
};

struct Spread {  // the tile shape of a product, and the workgroups of a tile
  int size, split;
};

// A tile's rows along m, and tokens (or rows) along n.
int tile_m(const Plan& k, int size) { return size == kDirect ? 32 : k.f32 ? (size == kBig ? 128 : 64) : size == kBig ? 256 : 128; }
int tile_n(const Plan& k, int size) { return size == kDirect ? 32 : !k.f32 && size == kBig ? 256 : 128; }

// The tile shape of the logits: large where such tiles fill the card, direct
// for a few tokens or few tiles.  Two accumulators of 16-bit types leave room
// for 256 x 128 at most, and two workgroups of 128 x 128 on a CU, which do not
// wait for each other, are faster (4096 x 1024 x 16384 bf16: 391 and 354 us).
int logits_size(const Plan& k, bool dual, int M, int N) {
  const auto tiles = [&](int size) { return cdiv(M, tile_m(k, size)) * cdiv(N, tile_n(k, size)); };
  if (N <= 32 || tiles(kSmall) < 96) return kDirect;
  if (dual && !k.f32) return kSmall;
  return tiles(kBig) >= (k.f32 ? 512 : 192) ? kBig : kSmall;
}

// Rows of parts that launch_logits writes for M vocabulary rows: one for each
// of the two waves that share a tile's.
int parts_of(const Plan& k, bool dual, int M, int N) {
  const int size = logits_size(k, dual, M, N);
  return (int)cdiv(M, tile_m(k, size)) * 2;
}

// Rows of parts that are kept before they are merged.
int max_parts(const Plan& k) {
  const int64_t n = kPartBytes / (8ll * k.N);
  return (int)(n < 4 ? 4 : n > 16384 ? 16384 : n);
}

// The vocabulary's pieces.  As few as the bounds allow: a piece's tiles are
// rounded up to whole rounds of the card (forward of 4096 x 1024 x 50001 bf16:
// 13 rounds in one piece, 14 in two; 409 us, 1030 TFLOP/s).
Plan plan_of(const ttt_lce_problem* p, int entry) {
  Plan k;
  k.dtype = p->dtype;
  k.entry = entry;
  k.f32 = p->dtype == TTT_F32;
  k.es = k.f32 ? 4 : 2;
  k.N = (int)p->rows;
  k.V = (int)p->vocab;
  k.d = (int)p->cols;
  k.dp = round8(k.d);
  k.pack = !k.f32 && k.d % 8 != 0;
  int64_t vc = kPieceRows;
  const auto bound = [&](int64_t rows) {
    if (rows < vc) vc = rows;
  };
  if (k.pack) bound(kPackBytes / ((int64_t)k.dp * 2));
  if (entry != TTT_LCE_FWD) bound(kPieceBytes / ((int64_t)k.N * k.es * (entry == TTT_LCE_BWD ? 1 : 2)));
  if (entry != TTT_LCE_BWD)
    while (vc > 256 && parts_of(k, entry == TTT_LCE_GG, (int)vc, k.N) > max_parts(k)) vc /= 2;
  vc = vc / 256 * 256;
  if (vc < 256) vc = 256;
  if (vc > p->vocab) vc = p->vocab;
  k.pieces = (int)cdiv(p->vocab, vc);
  vc = cdiv(cdiv(p->vocab, k.pieces), 256) * 256;
  if (vc > p->vocab) vc = p->vocab;
  k.vc = (int)vc;
  k.pieces = (int)cdiv(p->vocab, vc);
  return k;
}

// The tile shape and split of a plain product of k in `segs` segments: the
// least of (rounds of workgroups) x (steps of each) x (a step's time), plus the
// parts' traffic where they are split.  Steps (us) at full occupancy, measured
// on products that fill the card.
Spread spread_of(const Plan& p, int M, int N, int64_t k, bool keep) {
  const int step = p.f32 ? 32 : 64;
  const int steps = (int)cdiv(k, step);
  Spread best{kSmall, 1};
  double least = 1e30;
  for (int size = kSmall; size <= kBig; ++size) {
    const int slots = size == kBig ? 256 : 512;
    const double us = p.f32 ? (size == kBig ? 1.5 : 1.7) : size == kBig ? 1.75 : 1.25;
    const int64_t tiles = cdiv(M, tile_m(p, size)) * cdiv(N, tile_n(p, size));
    for (int split = 1; split <= kMaxSplit; split += split < 8 ? 1 : split < 24 ? 2 : 8) {
      if (split > 1 && split * 4 > steps) break;
      const int chunk = (int)cdiv(steps, split);
      const double rounds = (double)cdiv(tiles * split, slots);
      double t = rounds * (chunk * us + 3);
      if (split > 1 || keep) t += 4 + 8.0 * split * M * N / 4e6;
      if (t < least) {
        least = t;
        best = Spread{size, (int)cdiv(steps, chunk)};
      }
    }
  }
  return best;
}

// Of the products over a piece's vocabulary, [N, d], and over the tokens,
// [vc, d], with `segs` segments.
Spread spread_x(const Plan& k, int segs, bool keep) { return spread_of(k, k.d, k.N, (int64_t)segs * k.vc, keep); }
Spread spread_w(const Plan& k, int segs) { return spread_of(k, k.d, k.vc, (int64_t)segs * k.N, false); }

struct Buffers {
  void *xr, *ar, *wr, *br;  // row copies
  void *g, *hh;
  float *part_x, *part_w;  // fp32 parts of dx, dw
  float2 *part, *sums;
  float *at_target, *row, *h, *q, *coef, *live, *colmul, *rest_g, *rest_h, *alpha, *nx, *na, *nw, *nb;
  int parts;
};

// The same layout whatever outputs and cotangents a call has: sized for all.
Buffers layout(const Plan& k, Carver* c) {
  Buffers b;
  memset(&b, 0, sizeof(b));
  const bool fwd = k.entry == TTT_LCE_FWD, gg = k.entry == TTT_LCE_GG;
  if (fwd || gg) {
    const int whole = parts_of(k, gg, k.vc, k.N), last = parts_of(k, gg, k.V - (k.pieces - 1) * k.vc, k.N);
    const int64_t all = (int64_t)whole * (k.pieces - 1) + last;
    b.parts = all <= max_parts(k) ? (int)all : max_parts(k) + (whole > last ? whole : last);
  }
  if (b.parts) b.part = (float2*)c->take((int64_t)b.parts * k.N * 8);
  b.at_target = c->floats(k.N);
  b.row = c->floats(k.N);
  if (fwd) b.sums = (float2*)c->take(cdiv(k.N, 64) * 8);
  if (!k.f32) {
    const int64_t xb = 2 * (int64_t)k.N * k.dp;
    if (k.pack || !fwd) b.xr = c->take(xb);
    if (gg) b.ar = c->take(xb);
    if (k.pack) {
      b.wr = c->take(2 * (int64_t)k.vc * k.dp);
      if (gg) b.br = c->take(2 * (int64_t)k.vc * k.dp);
    }
  }
  if (fwd) return b;
  b.h = c->floats(k.N);
  b.q = c->floats(k.N);
  b.rest_g = c->floats(k.N);
  b.rest_h = c->floats(k.N);
  b.coef = c->floats(k.N);
  b.live = c->floats(k.N);
  b.colmul = c->floats(k.N);
  b.alpha = c->floats(1);
  const int64_t gb = (int64_t)k.es * k.N * piece_ld(k.vc);
  b.g = c->take(gb);
  if (gg) {
    b.hh = c->take(gb);
    if (k.dtype == TTT_F16) {
      b.nx = c->floats(k.N);
      b.na = c->floats(k.N);
      b.nw = c->floats(k.V);
      b.nb = c->floats(k.V);
    }
  }
  // parts: the most that any set of segments asks for; a product that is not
  // split and not added to needs none
  int64_t px = 0, pw = 0;
  const bool many = k.pieces > 1;
  for (int n = 1; n <= (gg ? 2 : 1); ++n) {
    for (int keep = many; keep <= (many || gg); ++keep) {
      const int s = spread_x(k, n, keep).split;
      if ((keep || s > 1) && s > px) px = s;
    }
    const int s = spread_w(k, n).split;
    if (s > 1 && s > pw) pw = s;
  }
  b.part_x = c->floats(px * k.N * k.d);
  b.part_w = c->floats(pw * k.vc * k.d);
  return b;
}

struct Operand {
  const void* p;
  int64_t ld;
};

void add_product(SegList* l, Operand m, Operand n, int k) {
  Seg& s = l->s[l->n++];
  s.m = m.p;
  s.n = n.p;
  s.ldm = m.ld;
  s.ldn = n.ld;
  s.k = k;
}

void launch_copy(const void* src, int64_t ld, int R, int C, void* dst, const float* live, hipStream_t st) {
  k_copy_rows<<<(unsigned)cdiv(R, 4), 256, 0, st>>>(CopyArgs{src, ld, R, C, dst, live});
}

template <int MODE>
void launch_logits(const Plan& k, ZArgs a, hipStream_t st) {
  constexpr bool dual = MODE >= kHSum;
  const int size = logits_size(k, dual, a.M, a.N);
  a.tm = (int)cdiv(a.M, tile_m(k, size));
  a.tn = (int)cdiv(a.N, tile_n(k, size));
  const unsigned grid = (unsigned)(a.tm * a.tn);
#define LOGITS(T)                                                                     \
  do {                                                                                \
    if (size == kDirect) {                                                            \
      k_logits<T, MODE, kDirect><<<grid, 256, 0, st>>>(a);                            \
      break;                                                                          \
    }                                                                                 \
    if constexpr (!dual || sizeof(T) == 4) {                                          \
      if (size == kBig) {                                                             \
        k_logits<T, MODE, kBig><<<grid, 512, 0, st>>>(a);                             \
        break;                                                                        \
      }                                                                               \
    }                                                                                 \
    k_logits<T, MODE, kSmall><<<grid, 256, 0, st>>>(a);                               \
  } while (0)
  if (k.dtype == TTT_F32) LOGITS(float);
  else if (k.dtype == TTT_BF16) LOGITS(__bf16);
  else LOGITS(_Float16);
#undef LOGITS
}

// Makes room in part for the rows of a piece of m vocabulary rows.
template <bool STATS>
void make_room(const Plan& k, const Buffers& b, int m, int* parts, hipStream_t st) {
  if (*parts + parts_of(k, !STATS, m, k.N) <= b.parts) return;
  k_merge<STATS><<<(unsigned)cdiv(k.N, 64), 1024, 0, st>>>(b.part, *parts, k.N);
  *parts = 1;
}

template <typename T>
void launch_product_of(const OutArgs& a, bool nt, int size, bool fin, hipStream_t st) {
  const unsigned grid = (unsigned)(a.tm * a.tn * a.split);
  if (size == kBig) {
    if (nt) k_product<T, true, kBig><<<grid, 512, 0, st>>>(a);
    else k_product<T, false, kBig><<<grid, 512, 0, st>>>(a);
  } else {
    if (nt) k_product<T, true, kSmall><<<grid, 256, 0, st>>>(a);
    else k_product<T, false, kSmall><<<grid, 256, 0, st>>>(a);
  }
  if (fin) k_finish<T><<<(unsigned)cdiv((int64_t)a.N * a.M, 1024), 256, 0, st>>>(a);
}

// One product (nt: its N operand is turned; the M operand always is).  keep:
// its fp32 parts stay (a later piece adds to them).  s: the spread of a whole
// piece's product, which the layout has room for; a shorter last piece has the
// same split (its own could be larger, and its parts past the room).
void launch_product(const Plan& k, OutArgs a, bool nt, float* part, bool keep, const Spread& s, bool last,
                    hipStream_t st) {
  int steps = 0;
  for (int i = 0; i < a.l.n; ++i) steps += (int)cdiv(a.l.s[i].k, k.f32 ? 32 : 64);
  a.tm = (int)cdiv(a.M, tile_m(k, s.size));
  a.tn = (int)cdiv(a.N, tile_n(k, s.size));
  a.split = s.split;
  a.chunk = (int)cdiv(steps, s.split);
  a.part = keep || s.split > 1 ? part : nullptr;
  const bool fin = a.part && last;
  if (k.dtype == TTT_F32) launch_product_of<float>(a, nt, s.size, fin, st);
  else if (k.dtype == TTT_BF16) launch_product_of<__bf16>(a, nt, s.size, fin, st);
  else launch_product_of<_Float16>(a, nt, s.size, fin, st);
}

int check(const ttt_lce_problem* p) {
  if (!p) return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: null problem");
  if (p->dtype != TTT_F16 && p->dtype != TTT_BF16 && p->dtype != TTT_F32)
    return ops_fail(TTT_ERR_UNSUPPORTED, "linear cross entropy: dtype code %d is not f16/bf16/f32", p->dtype);
  if (p->reduction < TTT_REDUCE_NONE || p->reduction > TTT_REDUCE_MEAN)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: reduction %d is not none, sum or mean",
                    p->reduction);
  if (p->rows < 1 || p->rows > 1 << 22 || p->vocab < 1 || p->vocab > 1 << 22)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: %lld rows, vocabulary %lld: each 1 .. 2^22",
                    (long long)p->rows, (long long)p->vocab);
  if (p->cols < 1 || p->cols > 1 << 16)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: rows of %lld values: 1 .. 2^16",
                    (long long)p->cols);
  return TTT_OK;
}

int take(const ttt_lce_problem* p, const ttt_rows* r, const char* name, bool need, bool operand) {
  if (!r || !r->data)
    return need ? ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: %s: null pointer", name) : TTT_OK;
  if (r->stride < p->cols || r->stride > 1 << 22)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: %s: row stride %lld: %lld .. 2^22", name,
                    (long long)r->stride, (long long)p->cols);
  const uintptr_t at = (uintptr_t)r->data;
  if (operand && p->dtype != TTT_F32 && p->cols % 8 == 0 && (at % 16 != 0 || r->stride % 8 != 0))
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: %s: rows not 16-byte aligned", name);
  if (at % (p->dtype == TTT_F32 ? 4 : 2))
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: %s: base pointer not aligned to its type", name);
  return TTT_OK;
}

#define TRY(x)                     \
  do {                             \
    const int rc_ = (x);           \
    if (rc_ != TTT_OK) return rc_; \
  } while (0)

int workspace(const Plan& k, void* ws, int64_t bytes, const char* what, Buffers* b) {
  Carver need{nullptr, 0};
  (void)layout(k, &need);
  if (!ws || bytes < need.used)
    return ops_fail(TTT_ERR_WORKSPACE, "%s: workspace of %lld bytes, needs %lld", what, ws ? (long long)bytes : 0ll,
                    (long long)need.used);
  if ((uintptr_t)ws % 16) return ops_fail(TTT_ERR_INVALID_ARGUMENT, "%s: workspace not 16-byte aligned", what);
  Carver c{(char*)ws, 0};
  *b = layout(k, &c);
  return TTT_OK;
}

int finish(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return ops_fail(TTT_ERR_LAUNCH, "%s: launch failed: %s", what, hipGetErrorString(e));
  return TTT_OK;
}

RowArgs row_args(const ttt_lce_problem* p, const Plan& k, const Buffers& b, const int64_t* target,
                 const float* weight, const float* row_stats, const float* grad_loss) {
  RowArgs r;
  memset(&r, 0, sizeof(r));
  r.N = k.N;
  r.V = k.V;
  r.reduction = p->reduction;
  r.dtype = k.dtype;
  r.ignore = p->ignore_index;
  r.target = target;
  r.weight = weight;
  r.stat = const_cast<float*>(row_stats);
  r.grad_loss = grad_loss;
  r.part = b.part;
  r.at_target = b.at_target;
  r.sums = b.sums;
  r.h = b.h;
  r.q = b.q;
  r.coef = b.coef;
  r.live = b.live;
  r.colmul = b.colmul;
  r.alpha = b.alpha;
  return r;
}

void launch_factors(const RowArgs& r, hipStream_t st) {
  k_factors<<<r.dtype == TTT_F32 ? (unsigned)cdiv(r.N, 1024) : 1, 1024, 0, st>>>(r);
}

// Rows v0 .. v0 + rows - 1 of an operand over d: copied, or as they are.
Operand rows_of(const Plan& k, const ttt_rows* w, int v0, int rows, void* copy, bool fresh, hipStream_t st) {
  const char* at = (const char*)w->data + (int64_t)v0 * w->stride * k.es;
  if (!k.pack) return {at, w->stride};
  if (fresh) launch_copy(at, w->stride, rows, k.d, copy, nullptr, st);
  return {copy, k.dp};
}

// X (or A) with zeros in the rows that do not count, where a sum over the rows will
// meet them (fp32: k_product leaves them out itself).
Operand live_rows(const Plan& k, const ttt_rows* x, void* copy, bool sums, const float* live, hipStream_t st) {
  if (k.f32 || (!k.pack && !sums)) return {x->data, x->stride};
  launch_copy(x->data, x->stride, k.N, k.d, copy, live, st);
  return {copy, k.dp};
}

// What the products of a call have in common.
struct Call {
  const Plan& k;
  const Buffers& b;
  hipStream_t st;

  // z (and u) tiles of vocabulary rows v0 .. v0 + m - 1
  ZArgs tiles(int v0, int m, const int64_t* target, const float* stat) const {
    ZArgs a;
    memset(&a, 0, sizeof(a));
    a.M = m;
    a.N = k.N;
    a.v0 = v0;
    a.target = target;
    a.stat = stat;
    a.h = b.h;
    a.q = b.q;
    a.colmul = b.colmul;
    a.rest_g = b.rest_g;
    a.rest_h = b.rest_h;
    return a;
  }
  // Operands that are G or H of a piece of m rows
  Operand piece(const void* g, int m) const { return {g, piece_ld(m)}; }

  // out [N, d] (+)= the list's product over the piece
  void over_vocab(const SegList& l, const ttt_rows* out, float* out32, bool add, bool keep, bool last,
                  const Rest& rest) const {
    OutArgs o;
    memset(&o, 0, sizeof(o));
    o.l = l;
    o.M = k.d;
    o.N = k.N;
    if (out) {
      o.out = out->data;
      o.ld = out->stride;
    }
    o.out32 = out32;
    o.rows = b.live;
    o.rest = rest;
    o.alpha = b.alpha;
    o.add = add;
    launch_product(k, o, false, b.part_x, keep, spread_x(k, l.n, keep), last, st);
  }
  // out rows v0 .. [m, d] = the list's product over the tokens
  void over_rows(const SegList& l, const ttt_rows* out, int v0, int m) const {
    OutArgs o;
    memset(&o, 0, sizeof(o));
    o.l = l;
    o.M = k.d;
    o.N = m;
    o.out = (char*)out->data + (int64_t)v0 * out->stride * k.es;
    o.ld = out->stride;
    o.live = k.f32 ? b.live : nullptr;
    o.alpha = b.alpha;
    launch_product(k, o, true, b.part_w, false, spread_w(k, l.n), true, st);
  }
};

bool given(const ttt_rows* r) { return r && r->data; }

}  // namespace
}  // namespace ttt

using namespace ttt;

extern "C" {

int64_t ttt_lce_workspace_size(const ttt_lce_problem* p, int32_t entry) {
  if (check(p) != TTT_OK) return -1;
  if (entry < TTT_LCE_FWD || entry > TTT_LCE_GG) {
    ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: entry %d", entry);
    return -1;
  }
  Carver c{nullptr, 0};
  (void)layout(plan_of(p, entry), &c);
  return c.used;
}

int ttt_lce_fwd(const ttt_lce_problem* p, const ttt_rows* x, const ttt_rows* w, const int64_t* target,
                const float* row_weight, float* loss, float* row_stats, void* ws, int64_t ws_bytes, void* stream) {
  TRY(check(p));
  TRY(take(p, x, "hidden", true, true));
  TRY(take(p, w, "weight", true, true));
  if (!target || !loss || !row_stats)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: target, loss and row_stats are needed");
  const Plan k = plan_of(p, TTT_LCE_FWD);
  Buffers b;
  TRY(workspace(k, ws, ws_bytes, "ttt_lce_fwd", &b));
  const hipStream_t st = (hipStream_t)stream;
  const Call call{k, b, st};
  const Operand xo = rows_of(k, x, 0, k.N, b.xr, true, st);
  int parts = 0;
  for (int v0 = 0; v0 < k.V; v0 += k.vc) {
    const int m = k.V - v0 < k.vc ? k.V - v0 : k.vc;
    ZArgs a = call.tiles(v0, m, target, nullptr);
    add_product(&a.z, rows_of(k, w, v0, m, b.wr, true, st), xo, k.f32 ? k.d : k.dp);
    make_room<true>(k, b, m, &parts, st);
    a.part = b.part + (int64_t)parts * k.N;
    a.at_target = b.at_target;
    launch_logits<kStats>(k, a, st);
    parts += parts_of(k, false, m, k.N);
  }
  RowArgs r = row_args(p, k, b, target, row_weight, row_stats, nullptr);
  r.parts = parts;
  r.row = p->reduction == TTT_REDUCE_NONE ? loss : b.row;
  r.out = loss;
  k_join_loss<<<(unsigned)cdiv(k.N, 64), 1024, 0, st>>>(r);
  if (k.N > 64 && p->reduction != TTT_REDUCE_NONE) k_reduce_loss<<<1, 1024, 0, st>>>(r);
  return finish("ttt_lce_fwd");
}

int ttt_lce_bwd(const ttt_lce_problem* p, const ttt_rows* x, const ttt_rows* w, const int64_t* target,
                const float* row_weight, const float* row_stats, const float* grad_loss, const ttt_rows* dx,
                const ttt_rows* dw, float* dx32, void* ws, int64_t ws_bytes, void* stream) {
  TRY(check(p));
  TRY(take(p, x, "hidden", true, true));
  TRY(take(p, w, "weight", true, true));
  TRY(take(p, dx, "dx", false, false));
  TRY(take(p, dw, "dw", false, false));
  if (!target || !row_stats || !grad_loss)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: target, row_stats and grad_loss are needed");
  const bool want_x = given(dx), want_w = given(dw);
  if (dx32 && !want_x) return ops_fail(TTT_ERR_INVALID_ARGUMENT, "ttt_lce_bwd: dx32 without dx");
  if (!want_x && !want_w) return TTT_OK;
  const Plan k = plan_of(p, TTT_LCE_BWD);
  Buffers b;
  TRY(workspace(k, ws, ws_bytes, "ttt_lce_bwd", &b));
  const hipStream_t st = (hipStream_t)stream;
  const Call call{k, b, st};
  launch_factors(row_args(p, k, b, target, row_weight, row_stats, grad_loss), st);
  const Operand xo = live_rows(k, x, b.xr, want_w, b.live, st);
  for (int v0 = 0; v0 < k.V; v0 += k.vc) {
    const int m = k.V - v0 < k.vc ? k.V - v0 : k.vc;
    const Operand wo = rows_of(k, w, v0, m, b.wr, true, st), go = call.piece(b.g, m);
    ZArgs a = call.tiles(v0, m, target, row_stats);
    add_product(&a.z, wo, xo, k.f32 ? k.d : k.dp);
    a.g = b.g;
    launch_logits<kGrad>(k, a, st);
    if (want_x) {
      SegList l{};
      add_product(&l, wo, go, m);
      call.over_vocab(l, dx, dx32, v0 > 0, k.pieces > 1, v0 + m >= k.V,
                      Rest{target, k.V, w->data, nullptr, w->stride, 0, b.rest_g, nullptr});
    }
    if (want_w) {
      SegList l{};
      add_product(&l, xo, go, k.N);
      call.over_rows(l, dw, v0, m);
    }
  }
  return finish("ttt_lce_bwd");
}

int ttt_lce_gg(const ttt_lce_problem* p, const ttt_rows* x, const ttt_rows* w, const int64_t* target,
               const float* row_weight, const float* row_stats, const float* grad_loss, const float* dx32,
               const ttt_rows* ca, const ttt_rows* cb, const ttt_rows* gx, const ttt_rows* gw, float* ggrad_loss,
               void* ws, int64_t ws_bytes, void* stream) {
  TRY(check(p));
  TRY(take(p, x, "hidden", true, true));
  TRY(take(p, w, "weight", true, true));
  TRY(take(p, ca, "a", false, true));
  TRY(take(p, cb, "b", false, true));
  TRY(take(p, gx, "gx", false, false));
  TRY(take(p, gw, "gw", false, false));
  if (!target || !row_stats || !grad_loss)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: target, row_stats and grad_loss are needed");
  const bool has_a = given(ca), has_b = given(cb), want_x = given(gx), want_w = given(gw);
  if (!has_a && !has_b)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "ttt_lce_gg: a cotangent of dx or of dw is needed");
  if (!want_x && !want_w && !ggrad_loss) return TTT_OK;
  const Plan k = plan_of(p, TTT_LCE_GG);
  Buffers b;
  TRY(workspace(k, ws, ws_bytes, "ttt_lce_gg", &b));
  const hipStream_t st = (hipStream_t)stream;
  const Call call{k, b, st};
  RowArgs r = row_args(p, k, b, target, row_weight, row_stats, grad_loss);
  if (k.dtype == TTT_F16) {
    NormList l{};
    int64_t rows = 0;
    const auto norms = [&](const ttt_rows* t, int n, float* out) {
      l.s[l.n++] = {t->data, t->stride, n, out};
      rows += n;
      return out;
    };
    l.cols = k.d;
    if (has_a) {
      r.na = norms(ca, k.N, b.na);
      r.nw = norms(w, k.V, b.nw);
    }
    if (has_b) {
      r.nx = norms(x, k.N, b.nx);
      r.nb = norms(cb, k.V, b.nb);
    }
    k_norms<_Float16><<<(unsigned)cdiv(rows, 4), 256, 0, st>>>(l);
  }
  launch_factors(r, st);
  const Operand xo = live_rows(k, x, b.xr, want_w, b.live, st);
  Operand ao{nullptr, 0};
  if (has_a) ao = live_rows(k, ca, b.ar, want_w, b.live, st);
  const int kd = k.f32 ? k.d : k.dp;
  const bool second = want_x || want_w;
  // h from dX and G B, or from its tiles
  const bool sums = ggrad_loss || (has_a && !dx32);
  const bool one = k.pieces == 1;  // a piece's copies and G last from the first walk to the second
  const auto zu = [&](int v0, int m, bool fresh, bool u) {
    ZArgs a = call.tiles(v0, m, target, row_stats);
    const Operand wo = rows_of(k, w, v0, m, b.wr, fresh, st);
    add_product(&a.z, wo, xo, kd);
    if (u && has_a) add_product(&a.u, wo, ao, kd);
    if (u && has_b) add_product(&a.u, rows_of(k, cb, v0, m, b.br, fresh, st), xo, kd);
    return a;
  };
  bool walked = false;
  if (sums) {
    int parts = 0;
    for (int v0 = 0; v0 < k.V; v0 += k.vc) {
      const int m = k.V - v0 < k.vc ? k.V - v0 : k.vc;
      ZArgs a = zu(v0, m, true, true);
      make_room<false>(k, b, m, &parts, st);
      a.part = b.part + (int64_t)parts * k.N;
      a.at_target = b.at_target;
      launch_logits<kHSum>(k, a, st);
      parts += parts_of(k, true, m, k.N);
    }
    walked = true;
    r.parts = parts;
    r.row = ggrad_loss ? (p->reduction == TTT_REDUCE_NONE ? ggrad_loss : b.row) : nullptr;
    k_join_h<<<(unsigned)cdiv(k.N, 64), 1024, 0, st>>>(r);
    if (ggrad_loss && p->reduction != TTT_REDUCE_NONE) k_sum<<<1, 1024, 0, st>>>(b.row, k.N, ggrad_loss);
  } else {
    HArgs h;
    memset(&h, 0, sizeof(h));
    if (has_b) {  // G B to the parts, where H W is added later
      for (int v0 = 0; v0 < k.V; v0 += k.vc) {
        const int m = k.V - v0 < k.vc ? k.V - v0 : k.vc;
        ZArgs a = zu(v0, m, true, false);
        a.g = b.g;
        launch_logits<kGrad>(k, a, st);
        SegList l{};
        add_product(&l, rows_of(k, cb, v0, m, b.br, true, st), call.piece(b.g, m), m);
        call.over_vocab(l, nullptr, nullptr, v0 > 0, true, false, Rest{});
      }
      walked = true;
      h.gb = b.part_x;
      h.split = spread_x(k, 1, true).split;
      h.rest = b.rest_g;
      h.b = cb->data;
      h.ldb = cb->stride;
    }
    if (has_a) {
      h.a = ca->data;
      h.lda = ca->stride;
      h.dx32 = dx32;
    }
    h.N = k.N;
    h.V = k.V;
    h.d = k.d;
    h.target = target;
    h.coef = b.coef;
    h.alpha = b.alpha;
    h.x = x->data;
    h.ldx = x->stride;
    h.w = w->data;
    h.ldw = w->stride;
    h.h = b.h;
    h.q = b.q;
    const unsigned grid = (unsigned)cdiv(k.N, 4);
    if (k.dtype == TTT_F32) k_row_h<float><<<grid, 256, 0, st>>>(h);
    else if (k.dtype == TTT_BF16) k_row_h<__bf16><<<grid, 256, 0, st>>>(h);
    else k_row_h<_Float16><<<grid, 256, 0, st>>>(h);
  }
  if (!second) return finish("ttt_lce_gg");
  const bool kept = !sums && has_b;  // G B waits in the parts
  for (int v0 = 0; v0 < k.V; v0 += k.vc) {
    const int m = k.V - v0 < k.vc ? k.V - v0 : k.vc;
    const bool fresh = !(walked && one);
    ZArgs a = zu(v0, m, fresh, true);
    const bool need_g = (want_x && has_b && sums) || (want_w && has_a);
    a.hh = b.hh;
    a.g = need_g && !(kept && one) ? b.g : nullptr;
    launch_logits<kHGrad>(k, a, st);
    const Operand go = call.piece(b.g, m), ho = call.piece(b.hh, m);
    if (want_x) {
      SegList l{};
      add_product(&l, rows_of(k, w, v0, m, b.wr, false, st), ho, m);
      if (has_b && sums) add_product(&l, rows_of(k, cb, v0, m, b.br, false, st), go, m);
      call.over_vocab(l, gx, nullptr, v0 > 0 || kept, k.pieces > 1 || kept, v0 + m >= k.V,
                      Rest{target, k.V, w->data, has_b ? cb->data : nullptr, w->stride, has_b ? cb->stride : 0,
                           b.rest_h, b.rest_g});
    }
    if (want_w) {
      SegList l{};
      add_product(&l, xo, ho, k.N);
      if (has_a) add_product(&l, ao, go, k.N);
      call.over_rows(l, gw, v0, m);
    }
  }
  return finish("ttt_lce_gg");
}

}  // extern "C"

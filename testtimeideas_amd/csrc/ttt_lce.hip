// ttt_lce.hip — the softmax cross entropy of a linear head for gfx950:
// forward, backward, double backward (formulas in include/ttt_ops.h), and
// their C entry points.
//
// Everything is tile products (ttt_gemm.h) with work done on the tiles where
// they are made:
//   forward    z tiles -> per tile and token (max, sum of exponentials)
//   backward   z tiles again -> p - 1_t, rounded once to the operand type, in
//              both orders; then dX = G W and dW = G^T X are plain products
//   gg         z and U tiles -> h = sum p U; again -> H (and G); then the
//              products [H|G][W;B] and [H^T|G^T][X;A]
// z is formed again instead of kept: 2 N V d operations against 4 N V bytes
// written and read.  G and H exist for one piece of the vocabulary at a time
// (pieces chosen to stay in the 256 MB last-level cache, kPieceBytes).
//
// fp32 problems run on the bf16 matrix cores: each operand is split into
// three bf16 parts whose sum is the value, and the six part products above
// 2^-24 of the whole are summed in fp32, smallest first.  G and H are split
// the same way where they are made.  An infinity becomes NaN this way.
//
// fp16 holds G and H scaled (kF16Scale, and per row by the largest |U|), since
// a softmax over a large vocabulary is below fp16's smallest values: powers
// of two, taken out again in fp32 when the products are stored.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/ttt_ops.h"
#include "ttt_gemm.h"
#include "ttt_ops.h"

namespace ttt {
namespace {

constexpr float kF16Scale = 16384.f;  // of a value in [-1, 1]: the largest power of two with room for sums

// Eight values to the parts of plane p (PL == 1: rounded to T; PL == 3: the
// p-th bf16 part of the fp32 value).
template <typename T, int PL>
__device__ __forceinline__ uint32_t part_pair(float a, float b, int p) {
  if constexpr (PL == 1) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    const t2 v = __builtin_convertvector(f32x2{a, b}, t2);
    uint32_t u;
    __builtin_memcpy(&u, &v, 4);
    return u;
  } else {
    uint32_t h, m, l;
    split_pair(a, b, h, m, l);
    return p == 0 ? h : p == 1 ? m : l;
  }
}

// ---------------------------------------------------------------------------
// Operand copies: rows padded to 8 columns, parts of fp32, transposes.
// ---------------------------------------------------------------------------
struct PackArgs {
  const void* src;       // [R, C], row stride ld
  int64_t ld;
  int R, C;
  void* rows;            // [PL][R][round8(C)], or null
  void* cols;            // [PL][C][round8(R)], or null
  const float* coef;     // rows whose factor is 0 are zeros in `cols`, or null
};

__host__ __device__ __forceinline__ int round8(int x) { return (x + 7) & ~7; }

// A 64 x 64 tile through LDS.
template <typename TS, typename T, int PL>
__global__ __launch_bounds__(256) void k_pack(PackArgs a) {
  __shared__ float tile[64][65];
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  const TS* src = (const TS*)a.src;
#pragma unroll 4
  for (int i = y; i < 64; i += 4) {
    const int r = r0 + i, c = c0 + x;
    tile[i][x] = r < a.R && c < a.C ? (float)src[(int64_t)r * a.ld + c] : 0.f;
  }
  __syncthreads();
  const int x2 = 2 * (threadIdx.x & 31), y2 = threadIdx.x >> 5;
  if (a.rows) {
    const int cp = round8(a.C);
    const int64_t plane = (int64_t)a.R * cp;
#pragma unroll 2
    for (int i = y2; i < 64; i += 8) {
      const int r = r0 + i, c = c0 + x2;
      if (r < a.R && c < cp)
#pragma unroll
        for (int p = 0; p < PL; ++p)
          *(uint32_t*)((uint16_t*)a.rows + p * plane + (int64_t)r * cp + c) =
              part_pair<T, PL>(tile[i][x2], tile[i][x2 + 1], p);
    }
  }
  if (a.cols) {
    const int rp = round8(a.R);
    const int64_t plane = (int64_t)a.C * rp;
    const bool in0 = r0 + x2 < a.R && (!a.coef || a.coef[r0 + x2] != 0.f);
    const bool in1 = r0 + x2 + 1 < a.R && (!a.coef || a.coef[r0 + x2 + 1] != 0.f);
#pragma unroll 2
    for (int i = y2; i < 64; i += 8) {
      const int c = c0 + i, r = r0 + x2;
      if (c < a.C && r < rp) {
        const float v0 = in0 ? tile[x2][i] : 0.f, v1 = in1 ? tile[x2 + 1][i] : 0.f;
#pragma unroll
        for (int p = 0; p < PL; ++p)
          *(uint32_t*)((uint16_t*)a.cols + p * plane + (int64_t)c * rp + r) = part_pair<T, PL>(v0, v1, p);
      }
    }
  }
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
  float2* part;       // [parts][N]: (max, sum) | (sum p U, max |U|)
  float* at_target;   // [N]: z or U at the target
  const float* h;     // [N]
  const float *rowmul, *colmul;
  void *grow, *gcol;  // p - 1_t: [PL][N][round8(M)], [PL][M][round8(N)]
  void *hrow, *hcol;  // p (U - h)
};

// The four-lane-group view of a wave's tile to a [n][m] matrix (rows) and to a
// [m][n] one (cols), through the wave's own 4 KB of LDS so that global stores
// are whole 128-byte rows.  val(i, j): the lane's four values of acc[i][j],
// 0 past M and N.
template <typename P, typename T, int PL, typename F>
__device__ __forceinline__ void store_rows(const P& tp, char* lds, void* out, int M, int N, F val) {
  constexpr int MI = P::MI, NI = P::NI, RB = MI * 32, CH = RB / 16;  // row bytes, chunks
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int ld = round8(M);
  const int64_t plane = (int64_t)N * ld;
  char* w = lds + 4096 * tp.wave;
  for (int p = 0; p < PL; ++p) {
    T* o = (T*)out + p * plane;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const f32x4 v = val(i, j);
        const u32x2 u = {part_pair<T, PL>(v[0], v[1], p), part_pair<T, PL>(v[2], v[3], p)};
        *(u32x2*)(w + c * RB + 16 * ((2 * i + (g >> 1)) ^ (c & 7)) + 8 * (g & 1)) = u;
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

template <typename P, typename T, int PL, typename F>
__device__ __forceinline__ void store_cols(const P& tp, char* lds, void* out, int M, int N, F val) {
  constexpr int MI = P::MI, NI = P::NI, RB = NI * 32, CH = RB / 16;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int ld = round8(N);
  const int64_t plane = (int64_t)M * ld;
  char* w = lds + 4096 * tp.wave;
  for (int p = 0; p < PL; ++p) {
    T* o = (T*)out + p * plane;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const f32x4 v = val(i, j);
        const uint32_t u0 = part_pair<T, PL>(v[0], v[1], p), u1 = part_pair<T, PL>(v[2], v[3], p);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          *(uint16_t*)(w + r * RB + 16 * ((2 * j + (c >> 3)) ^ (r & (CH - 1))) + 2 * (c & 7)) =
              (uint16_t)((e < 2 ? u0 : u1) >> (16 * (e & 1)));
        }
      }
#pragma unroll
      for (int t = 0; t < CH / 4; ++t) {
        const int r = t * (64 / CH) + lane / CH, ch = lane % CH;
        const u32x4 u = *(const u32x4*)(w + r * RB + 16 * (ch ^ (r & (CH - 1))));
        const int m = tp.m0 + (tp.wm * MI + i) * 16 + r, n = tp.n0 + tp.wn * NI * 16 + 8 * ch;
        if (m < M && n < ld) *(u32x4*)(o + (int64_t)m * ld + n) = u;
      }
    }
  }
}

template <typename T, int BM, int BN, int WM, int WN, int MODE, int PL>
__global__ __launch_bounds__(64 * WM * WN) void k_logits(ZArgs a) {
  typedef TileProduct<T, BM, BN, WM, WN> P;
  constexpr int MI = P::MI, NI = P::NI;
  constexpr bool kDual = MODE == kHSum || MODE == kHGrad;
  __shared__ __attribute__((aligned(16))) char sm0[BM * 128], sm1[BM * 128], sn0[BN * 128], sn1[BN * 128];
  static_assert(BM * 128 >= 4096 * WM * WN, "the epilogue's LDS");
  const typename P::Lds lds{sm0, sm1, sn0, sn1};
  int tm, tn;
  tile_of(blockIdx.x, a.tm, a.tn, &tm, &tn);
  P tp(tm * BM, tn * BN, a.M, a.N);
  f32x4 z[MI][NI], u[kDual ? MI : 1][kDual ? NI : 1];
  P::zero(z);
  tp.run(z, a.z, 0, a.z.steps, lds);
  if constexpr (kDual) {
    P::zero(u);
    tp.run(u, a.u, 0, a.u.steps, lds);
  }
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int n = tp.n_of(j);
    const bool nin = n < a.N;
    const int t = nin ? (int)(a.target[n] - a.v0) : -1;  // the target's row in the piece
    if constexpr (MODE == kStats) {
      float mx = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int m = tp.m_of(i) + e;
          if (m < a.M) mx = fmaxf(mx, z[i][j][e]);
          if (m == t && m < a.M) a.at_target[n] = z[i][j][e];
        }
      mx = group_max(mx);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s += tp.m_of(i) + e < a.M ? fast_exp2((z[i][j][e] - mx) * kLog2e) : 0.f;
      s = group_sum(s);
      if (g == 0 && nin) a.part[((int64_t)(tm * WM + tp.wm)) * a.N + n] = make_float2(mx, s);
    } else {
      const float mx = nin ? a.stat[n] : 0.f, inv = nin ? a.stat[a.N + n] : 0.f;
      const float h = MODE == kHGrad && nin ? a.h[n] : 0.f;
      float hs = 0.f, um = 0.f;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int m = tp.m_of(i) + e;
          const bool in = m < a.M && nin;
          const float p = in ? fast_exp2((z[i][j][e] - mx) * kLog2e) * inv : 0.f;
          if constexpr (kDual) {
            const float uu = u[i][j][e];
            if constexpr (MODE == kHSum) {
              hs += in ? p * uu : 0.f;
              um = fmaxf(um, in ? fabsf(uu) : 0.f);
              if (in && m == t) a.at_target[n] = uu;
            } else {
              u[i][j][e] = in ? p * (uu - h) : 0.f;
            }
          }
          z[i][j][e] = in && m == t ? p - 1.f : p;
        }
      if constexpr (MODE == kHSum) {
        hs = group_sum(hs);
        um = group_max(um);
        if (g == 0 && nin) a.part[((int64_t)(tm * WM + tp.wm)) * a.N + n] = make_float2(hs, um);
      }
    }
  }
  if constexpr (MODE == kGrad || MODE == kHGrad) {
    float rm[NI], cm[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int n = tp.n_of(j);
      rm[j] = n < a.N ? a.rowmul[n] : 0.f;
      cm[j] = n < a.N ? a.colmul[n] : 0.f;
    }
    // a row of factor 0 is 0 whatever its logits are
    if (a.grow) store_rows<P, T, PL>(tp, sm0, a.grow, a.M, a.N, [&](int i, int j) { return z[i][j] * rm[j]; });
    if (a.gcol)
      store_cols<P, T, PL>(tp, sm0, a.gcol, a.M, a.N, [&](int i, int j) {
        return cm[j] == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : z[i][j] * cm[j];
      });
    if constexpr (kDual) {
      if (a.hrow) store_rows<P, T, PL>(tp, sm0, a.hrow, a.M, a.N, [&](int i, int j) { return u[i][j] * rm[j]; });
      if (a.hcol)
        store_cols<P, T, PL>(tp, sm0, a.hcol, a.M, a.N, [&](int i, int j) {
          return cm[j] == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : u[i][j] * cm[j];
        });
    }
  }
}

// ---------------------------------------------------------------------------
// Plain products: out[n][m] = mul[n] * alpha * sum_k, to the output, or as
// fp32 to part[split][N][M] (added to what is there from earlier pieces).
// ---------------------------------------------------------------------------
struct OutArgs {
  SegList l;
  int M, N, tm, tn;
  int split, chunk;  // workgroups per tile, steps of each
  float* part;       // or null: direct
  int add;
  void* out;
  int64_t ld;
  const float* mul;    // [N] or null; a row of factor 0 is 0
  const float* alpha;  // one value or null
};

template <typename T, typename TO, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_product(OutArgs a) {
  typedef TileProduct<T, BM, BN, WM, WN> P;
  constexpr int MI = P::MI, NI = P::NI;
  __shared__ __attribute__((aligned(16))) char sm0[BM * 128], sm1[BM * 128], sn0[BN * 128], sn1[BN * 128];
  const typename P::Lds lds{sm0, sm1, sn0, sn1};
  const int s = blockIdx.x / (a.tm * a.tn), id = blockIdx.x % (a.tm * a.tn);
  int tm, tn;
  tile_of(id, a.tm, a.tn, &tm, &tn);
  P tp(tm * BM, tn * BN, a.M, a.N);
  f32x4 acc[MI][NI];
  P::zero(acc);
  const int lo = s * a.chunk, hi = lo + a.chunk < a.l.steps ? lo + a.chunk : a.l.steps;
  tp.run(acc, a.l, lo, hi, lds);
  const float al = a.part || !a.alpha ? 1.f : *a.alpha;
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int n = tp.n_of(j);
    if (n >= a.N) continue;
    const float mul = (a.part || !a.mul ? 1.f : a.mul[n]) * al;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = tp.m_of(i);
      if (m >= a.M) continue;
      f32x4 v = acc[i][j];
      if (a.part) {
        float* o = a.part + ((int64_t)s * a.N + n) * a.M + m;
        if (m + 4 <= a.M) {
          f32x4 old = {0.f, 0.f, 0.f, 0.f};
          if (a.add) __builtin_memcpy(&old, o, 16);
          v += old;
          __builtin_memcpy(o, &v, 16);
        } else {
          for (int e = 0; m + e < a.M; ++e) o[e] = a.add ? o[e] + v[e] : v[e];
        }
      } else {
        v = mul == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : v * mul;
        TO* o = (TO*)a.out + (int64_t)n * a.ld + m;
        if (m + 4 <= a.M) {
          TO r[4] = {(TO)v[0], (TO)v[1], (TO)v[2], (TO)v[3]};
          __builtin_memcpy(o, r, sizeof(r));
        } else {
          for (int e = 0; m + e < a.M; ++e) o[e] = (TO)v[e];
        }
      }
    }
  }
}

// out[n][m] = mul[n] * alpha * sum of the splits' parts, in their order.
template <typename TO>
__global__ __launch_bounds__(256) void k_finish(OutArgs a) {
  const int64_t total = (int64_t)a.N * a.M, i4 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i4 >= total) return;
  const float al = a.alpha ? *a.alpha : 1.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  const int cnt = total - i4 < 4 ? (int)(total - i4) : 4;
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
  for (int e = 0; e < cnt; ++e) {
    const int64_t n = (i4 + e) / a.M, m = (i4 + e) % a.M;
    const float mul = (a.mul ? a.mul[n] : 1.f) * al;
    ((TO*)a.out)[n * a.ld + m] = (TO)(mul == 0.f ? 0.f : v[e] * mul);
  }
}

// ---------------------------------------------------------------------------
// Row kernels.
// ---------------------------------------------------------------------------
struct RowArgs {
  int N, V, parts, reduction, f16;
  int64_t ignore;
  const int64_t* target;
  const float* weight;  // row weights or null
  const float2* part;
  const float* at_target;
  const float* grad_loss;
  float* stat;  // [2N + 2]: max, 1/sum, 1/denominator, weight sum
  float* row;   // [N]: the rows' losses | the rows' shares of the upstream gradient's gradient
  float* out;   // reduced
  float* h;
  float* umax;
  float *coef, *rowmul, *colmul, *outmul, *alpha;
};

__device__ __forceinline__ float row_weight(const RowArgs& a, int n) {
  return a.target[n] == a.ignore ? 0.f : a.weight ? a.weight[n] : 1.f;
}
__device__ __forceinline__ bool bad_target(const RowArgs& a, int n) { return a.target[n] < 0 || a.target[n] >= a.V; }

// The tiles' (max, sum) to the row's, and its loss: log(sum) - (z_t - max),
// which keeps its digits where the target has nearly all of the probability.
__global__ __launch_bounds__(256) void k_join_loss(RowArgs a) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= a.N) return;
  float mx = -__builtin_inff(), s = 0.f;
  for (int i = 0; i < a.parts; ++i) mx = fmaxf(mx, a.part[(int64_t)i * a.N + n].x);
  for (int i = 0; i < a.parts; ++i) {
    const float2 p = a.part[(int64_t)i * a.N + n];
    s += p.y == 0.f ? 0.f : p.y * fast_exp2((p.x - mx) * kLog2e);
  }
  a.stat[n] = mx;
  a.stat[a.N + n] = 1.f / s;
  const float w = row_weight(a, n);
  const float l = bad_target(a, n) ? __builtin_nanf("") : logf(s) - (a.at_target[n] - mx);
  a.row[n] = w == 0.f ? 0.f : w * l;
}

// Rows 0 .. parts - 1 of the tiles' partial results to row 0, so that what is
// kept does not grow with the vocabulary.
template <int MODE>
__global__ __launch_bounds__(256) void k_merge(float2* part, int parts, int N) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  if constexpr (MODE == kStats) {
    float mx = -__builtin_inff(), s = 0.f;
    for (int i = 0; i < parts; ++i) mx = fmaxf(mx, part[(int64_t)i * N + n].x);
    for (int i = 0; i < parts; ++i) {
      const float2 p = part[(int64_t)i * N + n];
      s += p.y == 0.f ? 0.f : p.y * fast_exp2((p.x - mx) * kLog2e);
    }
    part[n] = make_float2(mx, s);
  } else {
    float s = 0.f, um = 0.f;
    for (int i = 0; i < parts; ++i) {
      const float2 p = part[(int64_t)i * N + n];
      s += p.x;
      um = fmaxf(um, p.y);
    }
    part[n] = make_float2(s, um);
  }
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

// One workgroup: the rows' losses and weights to the loss and its denominator.
__global__ __launch_bounds__(1024) void k_reduce_loss(RowArgs a) {
  __shared__ float lds[16];
  float l = 0.f, w = 0.f;
  if (a.reduction != TTT_REDUCE_NONE)
    for (int n = threadIdx.x; n < a.N; n += 1024) {
      l += a.row[n];
      w += row_weight(a, n);
    }
  l = block_sum(l, lds);
  w = block_sum(w, lds);
  if (threadIdx.x == 0) {
    const float inv = a.reduction == TTT_REDUCE_MEAN ? 1.f / fmaxf(w, 1.f) : 1.f;
    a.stat[2 * a.N] = inv;
    a.stat[2 * a.N + 1] = w;
    if (a.reduction != TTT_REDUCE_NONE) a.out[0] = l * inv;
  }
}

// The rows' coefficients c and the factors that G is stored with.  fp16: one
// workgroup, which finds the largest |c| (times the row's scale) first.
__global__ __launch_bounds__(1024) void k_factors(RowArgs a) {
  __shared__ float lds[16];
  const float inv = a.stat[2 * a.N];
  float top = 0.f;
  const int stride = gridDim.x * 1024;
  for (int n = blockIdx.x * 1024 + threadIdx.x; n < a.N; n += stride) {
    const float w = row_weight(a, n);
    const float up = a.grad_loss[a.reduction == TTT_REDUCE_NONE ? n : 0];
    const float c = w == 0.f ? 0.f : bad_target(a, n) ? __builtin_nanf("") : up * w * inv;
    a.coef[n] = c;
    if (!a.f16) {
      a.rowmul[n] = 1.f;
      a.colmul[n] = a.outmul[n] = c;
    } else {
      // |p (U - h)| <= 2 max |U|: a power of two that keeps it (and p) below kF16Scale
      int e = 0;
      if (a.umax) (void)frexpf(fmaxf(1.f, 2.f * a.umax[n]), &e);
      const float rm = ldexpf(kF16Scale, -e);
      a.rowmul[n] = rm;
      a.outmul[n] = c / rm;
      const float t = fabsf(c / rm);
      if (t < __builtin_inff()) top = fmaxf(top, t);
    }
  }
  if (!a.f16) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.alpha = 1.f;
    return;
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
  __syncthreads();
  for (int i = 0; i < 16; ++i) top = fmaxf(top, lds[i]);
  int e = 0;
  (void)frexpf(top, &e);
  e = top == 0.f ? 0 : e > 120 ? 120 : e < -120 ? -120 : e;
  // c 2^-e / rm <= 1: the largest stored |value| is the row's own bound
  for (int n = threadIdx.x; n < a.N; n += 1024) a.colmul[n] = ldexpf(a.coef[n], -e);
  if (threadIdx.x == 0) *a.alpha = ldexpf(1.f, e);
}

__global__ __launch_bounds__(256) void k_join_h(RowArgs a) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= a.N) return;
  float s = 0.f, um = 0.f;
  for (int i = 0; i < a.parts; ++i) {
    const float2 p = a.part[(int64_t)i * a.N + n];
    s += p.x;
    um = fmaxf(um, p.y);
  }
  a.h[n] = s;
  if (a.umax) a.umax[n] = um;
  if (a.row) {
    const float w = row_weight(a, n);
    a.row[n] = w == 0.f ? 0.f
               : bad_target(a, n) ? __builtin_nanf("")
                                  : w * a.stat[2 * a.N] * (s - a.at_target[n]);
  }
}

__global__ __launch_bounds__(1024) void k_sum(const float* x, int n, float* out) {
  __shared__ float lds[16];
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) s += x[i];
  s = block_sum(s, lds);
  if (threadIdx.x == 0) *out = s;
}

// ---------------------------------------------------------------------------
// Host: sizes, workspace layout, launches.
// ---------------------------------------------------------------------------
constexpr int64_t kPieceBytes = 128ll << 20;  // G (and H) of a piece, all orders and parts
constexpr int64_t kPackBytes = 256ll << 20;   // packed head rows of a forward piece
constexpr int kMaxSplit = 16;
constexpr int kMaxParts = 1024;    // rows of the tiles' partial results that are kept before they are merged
constexpr int kStatsRows = 32768;  // vocabulary rows of a forward piece: at most kMaxParts / 2 such rows

struct Plan {
  int dtype, entry, PL, N, V, d, dp, Np;
  bool f32, pack;  // pack: rows are copied (parts of fp32, or not a multiple of 8 columns)
  int vc, pieces;  // vocabulary rows of a piece
};

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

Plan plan_of(const ttt_lce_problem* p, int entry) {
  Plan k;
  k.dtype = p->dtype;
  k.entry = entry;
  k.f32 = p->dtype == TTT_F32;
  k.PL = k.f32 ? 3 : 1;
  k.N = (int)p->rows;
  k.V = (int)p->vocab;
  k.d = (int)p->cols;
  k.dp = round8(k.d);
  k.Np = round8(k.N);
  k.pack = k.f32 || k.d % 8 != 0;
  int64_t vc = kStatsRows;
  if (entry == TTT_LCE_FWD) {
    const int64_t fit = kPackBytes / ((int64_t)k.dp * k.PL * 2);
    if (k.pack && fit < vc) vc = fit;
  } else {
    vc = kPieceBytes / ((int64_t)k.Np * k.PL * 2 * (entry == TTT_LCE_BWD ? 2 : 4));
  }
  vc = vc / 256 * 256;
  if (vc < 256) vc = 256;
  if (vc > kStatsRows) vc = kStatsRows;
  if (vc > p->vocab) vc = p->vocab;
  k.pieces = (int)cdiv(p->vocab, vc);
  vc = cdiv(cdiv(p->vocab, k.pieces), 256) * 256;
  if (vc > p->vocab) vc = p->vocab;
  k.vc = (int)vc;
  k.pieces = (int)cdiv(p->vocab, vc);
  return k;
}

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

struct Spread {  // the tiles of a product and the workgroups of each
  bool big;
  int tm, tn, split, chunk;
};

Spread spread_of(int M, int N, int steps) {
  Spread s;
  s.big = cdiv(M, 256) * cdiv(N, 256) >= 192;
  const int b = s.big ? 256 : 128;
  s.tm = (int)cdiv(M, b);
  s.tn = (int)cdiv(N, b);
  const int64_t tiles = (int64_t)s.tm * s.tn, want = s.big ? 256 : 512;
  int64_t split = tiles >= want / 2 ? 1 : cdiv(want, tiles);
  if (split > kMaxSplit) split = kMaxSplit;
  if (split > steps / 4) split = steps / 4 < 1 ? 1 : steps / 4;
  s.chunk = (int)cdiv(steps, split);
  s.split = (int)cdiv(steps, s.chunk);
  return s;
}

int steps_of(int k) { return (k + kStepK - 1) / kStepK; }

struct Buffers {
  // operand copies
  void *xr, *xt, *ar, *at;  // x and a: rows, transposed
  void *wr, *wt, *br, *bt;  // of the piece of w and b
  void *grow, *gcol, *hrow, *hcol;
  float *part_x, *part_w;   // fp32 parts of dx, dw
  float2* part;
  float *at_target, *row, *h, *umax, *coef, *rowmul, *colmul, *outmul, *alpha;
  int parts;
};

// The same layout whatever outputs and cotangents a call has: sized for all.
Buffers layout(const Plan& k, Carver* c) {
  Buffers b;
  memset(&b, 0, sizeof(b));
  const int64_t e = 2 * k.PL;
  const int vcp = round8(k.vc);
  const bool fwd = k.entry == TTT_LCE_FWD, gg = k.entry == TTT_LCE_GG;
  const int64_t each = cdiv(k.vc, 128) * 2;
  if (fwd || gg) b.parts = (int)(each * k.pieces < kMaxParts ? each * k.pieces : kMaxParts);
  if (b.parts) b.part = (float2*)c->take((int64_t)b.parts * k.N * 8);
  b.at_target = c->floats(k.N);
  b.row = c->floats(k.N);
  if (k.pack) {
    b.xr = c->take(e * k.N * k.dp);
    b.wr = c->take(e * k.vc * k.dp);
    if (gg) {
      b.ar = c->take(e * k.N * k.dp);
      b.br = c->take(e * k.vc * k.dp);
    }
  }
  if (fwd) return b;
  b.h = c->floats(k.N);
  b.umax = c->floats(k.N);
  b.coef = c->floats(k.N);
  b.rowmul = c->floats(k.N);
  b.colmul = c->floats(k.N);
  b.outmul = c->floats(k.N);
  b.alpha = c->floats(1);
  b.xt = c->take(e * k.d * k.Np);
  b.wt = c->take(e * k.d * vcp);
  b.grow = c->take(e * k.N * vcp);
  b.gcol = c->take(e * k.vc * k.Np);
  if (gg) {
    b.at = c->take(e * k.d * k.Np);
    b.bt = c->take(e * k.d * vcp);
    b.hrow = c->take(e * k.N * vcp);
    b.hcol = c->take(e * k.vc * k.Np);
  }
  // parts: the most that any set of segments asks for
  const int terms = k.f32 ? 6 : 1, most = gg ? 2 : 1;
  int64_t px = 0, pw = 0;
  for (int n = 1; n <= most; ++n) {
    const Spread sx = spread_of(k.d, k.N, n * terms * steps_of(vcp));
    const Spread sw = spread_of(k.d, k.vc, n * terms * steps_of(k.Np));
    if (sx.split > px) px = sx.split;
    if (sw.split > pw) pw = sw.split;
  }
  b.part_x = c->floats(px * k.N * k.d);
  b.part_w = c->floats(pw * k.vc * k.d);
  return b;
}

// The products of parts of an fp32 product, smallest first: (m part, n part).
const int kTerms[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};

// Adds the product of two packed (or 16-bit) operands over k to the list.
void add_product(SegList* l, const Plan& pl, const void* m, int64_t ldm, int64_t planem, const void* n, int64_t ldn,
                 int64_t planen, int k) {
  const int terms = pl.f32 ? 6 : 1;
  for (int t = 0; t < terms; ++t) {
    const int pm = pl.f32 ? kTerms[t][0] : 0, pn = pl.f32 ? kTerms[t][1] : 0;
    Seg& s = l->s[l->n++];
    s.m = (const char*)m + 2 * planem * pm;
    s.n = (const char*)n + 2 * planen * pn;
    s.ldm = ldm;
    s.ldn = ldn;
    s.k = k;
    l->steps += steps_of(k);
  }
}

struct Operand {
  const void* p;
  int64_t ld, plane;
};

void launch_pack(const Plan& k, const void* src, int64_t ld, int R, int C, void* rows, void* cols, const float* coef,
                 hipStream_t st) {
  if (!rows && !cols) return;
  PackArgs a{src, ld, R, C, rows, cols, coef};
  // the padded columns of `rows` and rows of `cols` lie in the last tiles
  const dim3 grid((unsigned)cdiv(C, 64), (unsigned)cdiv(R, 64));
  if (k.dtype == TTT_F32) k_pack<float, __bf16, 3><<<grid, 256, 0, st>>>(a);
  else if (k.dtype == TTT_BF16) k_pack<__bf16, __bf16, 1><<<grid, 256, 0, st>>>(a);
  else k_pack<_Float16, _Float16, 1><<<grid, 256, 0, st>>>(a);
}

template <int MODE>
void launch_logits(const Plan& k, ZArgs a, hipStream_t st) {
  constexpr bool dual = MODE == kHSum || MODE == kHGrad;
  const bool big = !dual && cdiv(a.M, 256) * cdiv(a.N, 256) >= 192;
  const int b = big ? 256 : 128;
  a.tm = (int)cdiv(a.M, b);
  a.tn = (int)cdiv(a.N, b);
  const unsigned grid = (unsigned)(a.tm * a.tn);
#define LOGITS(T, PL)                                                              \
  do {                                                                             \
    if constexpr (!dual) {                                                         \
      if (big) {                                                                   \
        k_logits<T, 256, 256, 2, 4, MODE, PL><<<grid, 512, 0, st>>>(a);            \
        break;                                                                     \
      }                                                                            \
    }                                                                              \
    k_logits<T, 128, 128, 2, 2, MODE, PL><<<grid, 256, 0, st>>>(a);                \
  } while (0)
  if (k.dtype == TTT_F32) LOGITS(__bf16, 3);
  else if (k.dtype == TTT_BF16) LOGITS(__bf16, 1);
  else LOGITS(_Float16, 1);
#undef LOGITS
}

// Rows of parts that launch_logits writes for M vocabulary rows (two waves of
// a tile's vocabulary each).
int parts_of(bool dual, int M, int N) {
  const bool big = !dual && cdiv(M, 256) * cdiv(N, 256) >= 192;
  return (int)cdiv(M, big ? 256 : 128) * 2;
}

// Makes room in part for the rows of a piece of m vocabulary rows.
template <int MODE>
void make_room(const Buffers& b, int N, int m, int* parts, hipStream_t st) {
  if (*parts + parts_of(MODE == kHSum, m, N) <= b.parts) return;
  k_merge<MODE><<<(unsigned)cdiv(N, 256), 256, 0, st>>>(b.part, *parts, N);
  *parts = 1;
}

void launch_finish(const Plan& k, const OutArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)cdiv((int64_t)a.N * a.M, 1024);
  if (k.dtype == TTT_F32) k_finish<float><<<grid, 256, 0, st>>>(a);
  else if (k.dtype == TTT_BF16) k_finish<__bf16><<<grid, 256, 0, st>>>(a);
  else k_finish<_Float16><<<grid, 256, 0, st>>>(a);
}

// One product.  keep: its fp32 parts stay (a later piece adds to them), with
// the split of the first piece, whose steps are `full`.
void launch_product(const Plan& k, OutArgs a, float* part, bool keep, int full, bool last, hipStream_t st) {
  const Spread s = spread_of(a.M, a.N, full);
  a.tm = s.tm;
  a.tn = s.tn;
  a.split = s.split;
  a.chunk = (int)cdiv(a.l.steps, s.split);
  a.part = keep || s.split > 1 ? part : nullptr;
  const unsigned grid = (unsigned)(s.tm * s.tn * s.split);
#define PRODUCT(T, TO)                                                                     \
  do {                                                                                     \
    if (s.big) k_product<T, TO, 256, 256, 2, 4><<<grid, 512, 0, st>>>(a);                  \
    else k_product<T, TO, 128, 128, 2, 2><<<grid, 256, 0, st>>>(a);                        \
  } while (0)
  if (k.dtype == TTT_F32) PRODUCT(__bf16, float);
  else if (k.dtype == TTT_BF16) PRODUCT(__bf16, __bf16);
  else PRODUCT(_Float16, _Float16);
#undef PRODUCT
  if (a.part && last) launch_finish(k, a, st);
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
                 const float* weight) {
  RowArgs r;
  memset(&r, 0, sizeof(r));
  r.N = k.N;
  r.V = k.V;
  r.reduction = p->reduction;
  r.f16 = k.dtype == TTT_F16;
  r.ignore = p->ignore_index;
  r.target = target;
  r.weight = weight;
  r.part = b.part;
  r.at_target = b.at_target;
  r.coef = b.coef;
  r.rowmul = b.rowmul;
  r.colmul = b.colmul;
  r.outmul = b.outmul;
  r.alpha = b.alpha;
  return r;
}

// Rows v0 .. of w (or b) as an operand over d: packed, or as they are.
Operand rows_of(const Plan& k, const ttt_rows* w, int v0, int rows, void* packed) {
  if (k.pack) return {packed, k.dp, (int64_t)rows * k.dp};
  return {(const char*)w->data + (int64_t)v0 * w->stride * 2, w->stride, 0};
}
const void* row_at(const Plan& k, const ttt_rows* w, int v0) {
  return (const char*)w->data + (int64_t)v0 * w->stride * (k.f32 ? 4 : 2);
}

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
  if (k.pack) launch_pack(k, x->data, x->stride, k.N, k.d, b.xr, nullptr, nullptr, st);
  const Operand xo = rows_of(k, x, 0, k.N, b.xr);
  int parts = 0;
  for (int v0 = 0; v0 < k.V; v0 += k.vc) {
    const int m = k.V - v0 < k.vc ? k.V - v0 : k.vc;
    if (k.pack) launch_pack(k, row_at(k, w, v0), w->stride, m, k.d, b.wr, nullptr, nullptr, st);
    const Operand wo = rows_of(k, w, v0, m, b.wr);
    ZArgs a;
    memset(&a, 0, sizeof(a));
    add_product(&a.z, k, wo.p, wo.ld, wo.plane, xo.p, xo.ld, xo.plane, k.dp);
    a.M = m;
    a.N = k.N;
    a.v0 = v0;
    a.target = target;
    make_room<kStats>(b, k.N, m, &parts, st);
    a.part = b.part + (int64_t)parts * k.N;
    a.at_target = b.at_target;
    launch_logits<kStats>(k, a, st);
    parts += parts_of(false, m, k.N);
  }
  RowArgs r = row_args(p, k, b, target, row_weight);
  r.parts = parts;
  r.stat = row_stats;
  r.row = p->reduction == TTT_REDUCE_NONE ? loss : b.row;
  r.out = loss;
  k_join_loss<<<(unsigned)cdiv(k.N, 256), 256, 0, st>>>(r);
  k_reduce_loss<<<1, 1024, 0, st>>>(r);
  return finish("ttt_lce_fwd");
}

int ttt_lce_bwd(const ttt_lce_problem* p, const ttt_rows* x, const ttt_rows* w, const int64_t* target,
                const float* row_weight, const float* row_stats, const float* grad_loss, const ttt_rows* dx,
                const ttt_rows* dw, void* ws, int64_t ws_bytes, void* stream) {
  TRY(check(p));
  TRY(take(p, x, "hidden", true, true));
  TRY(take(p, w, "weight", true, true));
  TRY(take(p, dx, "dx", false, false));
  TRY(take(p, dw, "dw", false, false));
  if (!target || !row_stats || !grad_loss)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: target, row_stats and grad_loss are needed");
  const bool want_x = dx && dx->data, want_w = dw && dw->data;
  if (!want_x && !want_w) return TTT_OK;
  const Plan k = plan_of(p, TTT_LCE_BWD);
  Buffers b;
  TRY(workspace(k, ws, ws_bytes, "ttt_lce_bwd", &b));
  const hipStream_t st = (hipStream_t)stream;
  RowArgs r = row_args(p, k, b, target, row_weight);
  r.stat = const_cast<float*>(row_stats);
  r.grad_loss = grad_loss;
  k_factors<<<r.f16 ? 1 : (unsigned)cdiv(k.N, 1024), 1024, 0, st>>>(r);
  launch_pack(k, x->data, x->stride, k.N, k.d, k.pack ? b.xr : nullptr, want_w ? b.xt : nullptr, b.coef, st);
  const Operand xo = rows_of(k, x, 0, k.N, b.xr);
  int full = 0;
  for (int v0 = 0; v0 < k.V; v0 += k.vc) {
    const int m = k.V - v0 < k.vc ? k.V - v0 : k.vc, mp = round8(m);
    launch_pack(k, row_at(k, w, v0), w->stride, m, k.d, k.pack ? b.wr : nullptr, want_x ? b.wt : nullptr, nullptr, st);
    const Operand wo = rows_of(k, w, v0, m, b.wr);
    ZArgs a;
    memset(&a, 0, sizeof(a));
    add_product(&a.z, k, wo.p, wo.ld, wo.plane, xo.p, xo.ld, xo.plane, k.dp);
    a.M = m;
    a.N = k.N;
    a.v0 = v0;
    a.target = target;
    a.stat = row_stats;
    a.rowmul = b.rowmul;
    a.colmul = b.colmul;
    a.grow = want_x ? b.grow : nullptr;
    a.gcol = want_w ? b.gcol : nullptr;
    launch_logits<kGrad>(k, a, st);
    if (want_x) {
      OutArgs o;
      memset(&o, 0, sizeof(o));
      add_product(&o.l, k, b.wt, mp, (int64_t)k.d * mp, b.grow, mp, (int64_t)k.N * mp, mp);
      o.M = k.d;
      o.N = k.N;
      o.out = dx->data;
      o.ld = dx->stride;
      o.mul = b.outmul;
      o.add = v0 > 0;
      if (v0 == 0) full = o.l.steps;
      launch_product(k, o, b.part_x, k.pieces > 1, full, v0 + m >= k.V, st);
    }
    if (want_w) {
      OutArgs o;
      memset(&o, 0, sizeof(o));
      add_product(&o.l, k, b.xt, k.Np, (int64_t)k.d * k.Np, b.gcol, k.Np, (int64_t)m * k.Np, k.Np);
      o.M = k.d;
      o.N = m;
      o.out = (char*)dw->data + (int64_t)v0 * dw->stride * (k.f32 ? 4 : 2);
      o.ld = dw->stride;
      o.alpha = b.alpha;
      launch_product(k, o, b.part_w, false, o.l.steps, true, st);
    }
  }
  return finish("ttt_lce_bwd");
}

int ttt_lce_gg(const ttt_lce_problem* p, const ttt_rows* x, const ttt_rows* w, const int64_t* target,
               const float* row_weight, const float* row_stats, const float* grad_loss, const ttt_rows* ca,
               const ttt_rows* cb, const ttt_rows* gx, const ttt_rows* gw, float* ggrad_loss, void* ws,
               int64_t ws_bytes, void* stream) {
  TRY(check(p));
  TRY(take(p, x, "hidden", true, true));
  TRY(take(p, w, "weight", true, true));
  TRY(take(p, ca, "a", false, true));
  TRY(take(p, cb, "b", false, true));
  TRY(take(p, gx, "gx", false, false));
  TRY(take(p, gw, "gw", false, false));
  if (!target || !row_stats || !grad_loss)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "linear cross entropy: target, row_stats and grad_loss are needed");
  const bool has_a = ca && ca->data, has_b = cb && cb->data;
  const bool want_x = gx && gx->data, want_w = gw && gw->data;
  if (!has_a && !has_b)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "ttt_lce_gg: a cotangent of dx or of dw is needed");
  if (!want_x && !want_w && !ggrad_loss) return TTT_OK;
  const Plan k = plan_of(p, TTT_LCE_GG);
  Buffers b;
  TRY(workspace(k, ws, ws_bytes, "ttt_lce_gg", &b));
  const hipStream_t st = (hipStream_t)stream;
  RowArgs r = row_args(p, k, b, target, row_weight);
  r.stat = const_cast<float*>(row_stats);
  r.grad_loss = grad_loss;
  // c before the transposes (rows of factor 0 are left out of them); fp16's scales follow the first pass
  r.f16 = 0;
  k_factors<<<(unsigned)cdiv(k.N, 1024), 1024, 0, st>>>(r);
  launch_pack(k, x->data, x->stride, k.N, k.d, k.pack ? b.xr : nullptr, want_w ? b.xt : nullptr, b.coef, st);
  if (has_a)
    launch_pack(k, ca->data, ca->stride, k.N, k.d, k.pack ? b.ar : nullptr, want_w ? b.at : nullptr, b.coef, st);
  const Operand xo = rows_of(k, x, 0, k.N, b.xr);
  Operand ao{nullptr, 0, 0};
  if (has_a) ao = rows_of(k, ca, 0, k.N, b.ar);
  const bool second = want_x || want_w;
  int parts = 0, full = 0;
  for (int pass = 0; pass < (second ? 2 : 1); ++pass) {
    for (int v0 = 0; v0 < k.V; v0 += k.vc) {
      const int m = k.V - v0 < k.vc ? k.V - v0 : k.vc, mp = round8(m);
      const bool turned = pass == 1 && want_x;
      const bool fresh = pass == 0 || k.pieces > 1;  // one piece: the rows packed for the first pass are there
      launch_pack(k, row_at(k, w, v0), w->stride, m, k.d, k.pack && fresh ? b.wr : nullptr, turned ? b.wt : nullptr,
                  nullptr, st);
      if (has_b)
        launch_pack(k, row_at(k, cb, v0), cb->stride, m, k.d, k.pack && fresh ? b.br : nullptr,
                    turned ? b.bt : nullptr, nullptr, st);
      const Operand wo = rows_of(k, w, v0, m, b.wr);
      ZArgs a;
      memset(&a, 0, sizeof(a));
      add_product(&a.z, k, wo.p, wo.ld, wo.plane, xo.p, xo.ld, xo.plane, k.dp);
      if (has_a) add_product(&a.u, k, wo.p, wo.ld, wo.plane, ao.p, ao.ld, ao.plane, k.dp);
      if (has_b) {
        const Operand bo = rows_of(k, cb, v0, m, b.br);
        add_product(&a.u, k, bo.p, bo.ld, bo.plane, xo.p, xo.ld, xo.plane, k.dp);
      }
      a.M = m;
      a.N = k.N;
      a.v0 = v0;
      a.target = target;
      a.stat = row_stats;
      if (pass == 0) {
        make_room<kHSum>(b, k.N, m, &parts, st);
        a.part = b.part + (int64_t)parts * k.N;
        a.at_target = b.at_target;
        launch_logits<kHSum>(k, a, st);
        parts += parts_of(true, m, k.N);
        continue;
      }
      a.h = b.h;
      a.rowmul = b.rowmul;
      a.colmul = b.colmul;
      a.hrow = want_x ? b.hrow : nullptr;
      a.hcol = want_w ? b.hcol : nullptr;
      a.grow = want_x && has_b ? b.grow : nullptr;
      a.gcol = want_w && has_a ? b.gcol : nullptr;
      launch_logits<kHGrad>(k, a, st);
      if (want_x) {
        OutArgs o;
        memset(&o, 0, sizeof(o));
        add_product(&o.l, k, b.wt, mp, (int64_t)k.d * mp, b.hrow, mp, (int64_t)k.N * mp, mp);
        if (has_b) add_product(&o.l, k, b.bt, mp, (int64_t)k.d * mp, b.grow, mp, (int64_t)k.N * mp, mp);
        o.M = k.d;
        o.N = k.N;
        o.out = gx->data;
        o.ld = gx->stride;
        o.mul = b.outmul;
        o.add = v0 > 0;
        if (v0 == 0) full = o.l.steps;
      launch_product(k, o, b.part_x, k.pieces > 1, full, v0 + m >= k.V, st);
      }
      if (want_w) {
        OutArgs o;
        memset(&o, 0, sizeof(o));
        add_product(&o.l, k, b.xt, k.Np, (int64_t)k.d * k.Np, b.hcol, k.Np, (int64_t)m * k.Np, k.Np);
        if (has_a) add_product(&o.l, k, b.at, k.Np, (int64_t)k.d * k.Np, b.gcol, k.Np, (int64_t)m * k.Np, k.Np);
        o.M = k.d;
        o.N = m;
        o.out = (char*)gw->data + (int64_t)v0 * gw->stride * (k.f32 ? 4 : 2);
        o.ld = gw->stride;
        o.alpha = b.alpha;
        launch_product(k, o, b.part_w, false, o.l.steps, true, st);
      }
    }
    if (pass == 0) {
      r.parts = parts;
      r.h = b.h;
      r.umax = k.dtype == TTT_F16 ? b.umax : nullptr;
      r.row = ggrad_loss ? (p->reduction == TTT_REDUCE_NONE ? ggrad_loss : b.row) : nullptr;
      k_join_h<<<(unsigned)cdiv(k.N, 256), 256, 0, st>>>(r);
      if (ggrad_loss && p->reduction != TTT_REDUCE_NONE) k_sum<<<1, 1024, 0, st>>>(b.row, k.N, ggrad_loss);
      if (second && k.dtype == TTT_F16) {
        r.f16 = 1;
        k_factors<<<1, 1024, 0, st>>>(r);
      }
    }
  }
  return finish("ttt_lce_gg");
}

}  // extern "C"

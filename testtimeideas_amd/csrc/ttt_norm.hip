// ttt_norm.hip — layer norm for gfx950: forward, backward, double backward
// (formulas in include/ttt_ops.h), and their C entry points.
//
// All three move a few [rows, cols] tensors once and do some tens of
// operations per element: bound by HBM.  A row is held in registers between
// its loads and its stores, by one wave (short rows: no barrier at all) or by
// a workgroup, in 16-byte chunks; every mean is a sum over the row by lane
// swaps (and LDS across waves).  The row's own mean and variance are formed in
// two passes over the registers, so a large common offset costs no digits.
// Column sums (dw, db, gw) stay in registers while a workgroup walks its rows;
// the workgroups' fp32 sums are added in workgroup order by a second launch.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/ttt_ops.h"
#include "ttt_common.h"
#include "ttt_ops.h"

namespace ttt {
namespace {

struct NormArgs {
  const void *x, *dy, *a;          // [N, D]
  void *y, *gx;                    // outputs [N, D]: y | dx | gx, and gdy
  int64_t ldx, lddy, lda, ldy, ldgx;
  const void *w, *b;               // parameters, or the cotangents cw, cb
  const void *cw, *cb;
  float *mean, *rstd;
  float* part;                     // [groups][nsum][D]
  int N, D, wf32;
  float eps;
};

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// A chunk as it was loaded: eight 16-bit or four fp32 values.  The loads are 16
// bytes wide whatever the address is (global memory takes any); values past D
// read as 0.
template <typename T>
struct Raw {
  T v[kVec<T>];
};

template <typename T, bool WHOLE>
__device__ __forceinline__ Raw<T> load_raw(const T* row, int col, int D) {
  constexpr int V = kVec<T>;
  Raw<T> r;
  if (WHOLE ? col < D : col + V <= D) {
    __builtin_memcpy(r.v, row + col, 16);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = !WHOLE && col + j < D ? row[col + j] : (T)0.f;
  }
  return r;
}

template <typename T, bool WHOLE>
__device__ __forceinline__ void store_chunk(T* row, int col, int D, const float* v) {
  constexpr int V = kVec<T>;
  if (WHOLE ? col < D : col + V <= D) {
    T r[V];
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = (T)v[j];
    __builtin_memcpy(row + col, r, 16);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!WHOLE && col + j < D) row[col + j] = (T)v[j];
  }
}

// A chunk's parameters at column col: of type T, or fp32 (f32); `none` where p is null.
template <typename T, bool WHOLE>
__device__ __forceinline__ void load_param(const void* p, int f32, int col, int D, float none, float* v) {
  constexpr int V = kVec<T>;
  if (!p) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = none;
  } else if (f32) {
    const float* q = (const float*)p;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = col + j < D ? q[col + j] : 0.f;
  } else {
    const Raw<T> r = load_raw<T, WHOLE>((const T*)p, col, D);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)r.v[j];
  }
}

// Sum over a wave, to every lane: lane swaps within 16 lanes (DPP: pairs,
// halves of four, mirrored halves and rows), then across (group_sum).
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __uint_as_float(__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = dpp_add<0xB1>(x);   // quad_perm 1,0,3,2
  x = dpp_add<0x4E>(x);   // quad_perm 2,3,0,1
  x = dpp_add<0x141>(x);  // row_half_mirror
  x = dpp_add<0x140>(x);  // row_mirror
  return group_sum(x);
}

// Sums of NS values over the threads of a row (TPR = 64: a wave; more: the
// workgroup, through LDS, `turn` picking one of two places so that one barrier
// does), to every thread.
template <int TPR, int NS>
__device__ __forceinline__ void row_sums(float* s, float* lds, int turn) {
#pragma unroll
  for (int k = 0; k < NS; ++k) s[k] = wave_sum(s[k]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int w = threadIdx.x >> 6;
    lds += turn * (NS * W);
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < NS; ++k) lds[k * W + w] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) t += lds[k * W + i];
      s[k] = t;
    }
  }
}

// Thread's chunk `ch` of a row: columns in chunk-major order, so a wave's
// loads of one chunk are contiguous.
template <typename T, int TPR>
__device__ __forceinline__ int chunk_col(int ch) {
  return (ch * TPR + (int)(threadIdx.x % TPR)) * kVec<T>;
}

// The chunks of a row of x; rows past the last are not read.
template <typename T, int TPR, int NCH, bool WHOLE>
__device__ __forceinline__ void load_row(const void* x, int64_t ld, int64_t row, const NormArgs& a, Raw<T>* r) {
  if (row < a.N) {
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) r[ch] = load_raw<T, WHOLE>((const T*)x + row * ld, chunk_col<T, TPR>(ch), a.D);
  }
}

// WHOLE: rows are whole chunks.  The loads of a part of a chunk, value by value,
// take up to 32 registers, and rows in flight with them (8192 x 2048 bf16: gg
// 50 -> 39 us; forward, with the parameters loaded once, 27 -> 14 us).  Measured:
// 65536 x 4096 bf16 forward 208 us, backward 296 us, both at the 5.0 to 5.4 TB/s
// of a large copy; 8192 x 384 fp32 forward 9.4, backward 11.1, gg 18.1 us (a
// copy of as many bytes: 5, 8 and 13).
//
// Every kernel walks its rows with the next row's loads in flight while this
// row is reduced and stored.  Rows past 2^31 - 1 do not exist, but row + stride
// may pass that: 64-bit rows.
template <typename T, int TPR, int NCH, int THREADS, bool WHOLE>
__global__ __launch_bounds__(THREADS) void k_norm_fwd(NormArgs a) {
  constexpr int V = kVec<T>, R = THREADS / TPR;
  __shared__ float lds[2 * 2 * 16];
  const int64_t stride = (int64_t)gridDim.x * R;
  int64_t row = (int64_t)blockIdx.x * R + (int)threadIdx.x / TPR;
  const float inv = 1.f / (float)a.D;
  Raw<T> x[NCH];
  load_row<T, TPR, NCH, WHOLE>(a.x, a.ldx, row, a, x);
  float w[NCH][V], b[NCH][V];
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    load_param<T, WHOLE>(a.w, a.wf32, chunk_col<T, TPR>(ch), a.D, 1.f, w[ch]);
    load_param<T, WHOLE>(a.b, a.wf32, chunk_col<T, TPR>(ch), a.D, 0.f, b[ch]);
  }
  for (int turn = 0; row < a.N; row += stride, turn ^= 1) {
    float v[NCH][V], s[1] = {0.f};
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[ch][j] = (float)x[ch].v[j];
        s[0] += v[ch][j];
      }
    load_row<T, TPR, NCH, WHOLE>(a.x, a.ldx, row + stride, a, x);
    row_sums<TPR, 1>(s, lds, turn);
    const float mu = s[0] * inv;
    float q[1] = {0.f};
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[ch][j] -= mu;
        q[0] += c0 + j < a.D ? v[ch][j] * v[ch][j] : 0.f;
      }
    }
    row_sums<TPR, 1>(q, lds + 32, turn);
    const float r = 1.f / sqrtf(q[0] * inv + a.eps);
    if (a.mean && threadIdx.x % TPR == 0) {
      a.mean[row] = mu;
      a.rstd[row] = r;
    }
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      if (c0 >= a.D) break;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = v[ch][j] * r * w[ch][j] + b[ch][j];
      store_chunk<T, WHOLE>((T*)a.y + row * a.ldy, c0, a.D, y);
    }
  }
}

// The column sums of a workgroup's rows to part[group][k][D].  With TPR = 64
// the waves hold sums of the same columns: added through LDS in wave order.
template <typename T, int TPR, int NCH, int THREADS, bool WHOLE, int NSUM>
__device__ __forceinline__ void store_sums(const NormArgs& a, float (*acc)[NCH][kVec<T>], float* lds) {
  constexpr int V = kVec<T>, W = THREADS / TPR, COLS = 64 * V;
  float* part = a.part + (int64_t)blockIdx.x * NSUM * a.D;
#pragma unroll
  for (int k = 0; k < NSUM; ++k)
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      if constexpr (TPR == THREADS) {
        store_chunk<float, WHOLE>(part + (int64_t)k * a.D, c0, a.D, acc[k][ch]);
        if constexpr (V == 8) store_chunk<float, WHOLE>(part + (int64_t)k * a.D, c0 + 4, a.D, acc[k][ch] + 4);
      } else {
        const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) lds[w * COLS + j * 64 + lane] = acc[k][ch][j];
        __syncthreads();
        for (int i = threadIdx.x; i < COLS; i += THREADS) {
          const int j = i / 64, l = i % 64, col = (ch * 64 + l) * V + j;
          float t = 0.f;
#pragma unroll
          for (int u = 0; u < W; ++u) t += lds[u * COLS + i];
          if (col < a.D) part[(int64_t)k * a.D + col] = t;
        }
      }
    }
}

template <typename T, int TPR, int NCH, int THREADS, bool WHOLE>
__global__ __launch_bounds__(THREADS) void k_norm_bwd(NormArgs a) {
  constexpr int V = kVec<T>, R = THREADS / TPR;
  __shared__ float lds[TPR == THREADS ? 2 * 2 * 16 : R * 64 * V];
  float w[NCH][V], acc[2][NCH][V];
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    load_param<T, WHOLE>(a.w, a.wf32, chunk_col<T, TPR>(ch), a.D, 1.f, w[ch]);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[0][ch][j] = acc[1][ch][j] = 0.f;
  }
  const float inv = 1.f / (float)a.D;
  const int64_t stride = (int64_t)gridDim.x * R;
  int64_t row = (int64_t)blockIdx.x * R + (int)threadIdx.x / TPR;
  Raw<T> x[NCH], dy[NCH];
  load_row<T, TPR, NCH, WHOLE>(a.x, a.ldx, row, a, x);
  load_row<T, TPR, NCH, WHOLE>(a.dy, a.lddy, row, a, dy);
  for (int turn = 0; row < a.N; row += stride, turn ^= 1) {
    const float r = a.rstd[row], mr = -a.mean[row] * r;
    float xh[NCH][V], g[NCH][V], s[2] = {0.f, 0.f};
    // past D: dy reads 0 there, and so nothing of xh counts
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[ch][j] = (float)x[ch].v[j] * r + mr;
        g[ch][j] = (float)dy[ch].v[j];
        acc[0][ch][j] += g[ch][j] * xh[ch][j];
        acc[1][ch][j] += g[ch][j];
        g[ch][j] *= w[ch][j];
        s[0] += g[ch][j];
        s[1] += g[ch][j] * xh[ch][j];
      }
    load_row<T, TPR, NCH, WHOLE>(a.x, a.ldx, row + stride, a, x);
    load_row<T, TPR, NCH, WHOLE>(a.dy, a.lddy, row + stride, a, dy);
    if (!a.y) continue;  // uniform
    row_sums<TPR, 2>(s, lds, turn);
    const float m1 = -r * s[0] * inv, m2 = -r * s[1] * inv;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      if (c0 >= a.D) break;
#pragma unroll
      for (int j = 0; j < V; ++j) g[ch][j] = r * g[ch][j] + (m1 + xh[ch][j] * m2);
      store_chunk<T, WHOLE>((T*)a.y + row * a.ldy, c0, a.D, g[ch]);
    }
  }
  if (a.part) store_sums<T, TPR, NCH, THREADS, WHOLE, 2>(a, acc, lds);
}

// The sums of t = cw dy - r (a mean(g xh) + g mean(a xh)) and of a P(g) follow
// from seven sums over the row itself, taken at once:
//   sum t      = sum(cw dy)    - r (mean(g xh) sum a      + mean(a xh) sum g)
//   sum t xh   = sum(cw dy xh) - r (mean(g xh) sum(a xh) + mean(a xh) sum(g xh))
//   sum a P(g) = sum a g - mean(g) sum a - mean(g xh) sum(a xh)
// so there is one reduction, and about 25 operations per element (they are
// what bounds this kernel where its rows come from the cache).
template <typename T, int TPR, int NCH, int THREADS, bool WHOLE>
__global__ __launch_bounds__(THREADS) void k_norm_gg(NormArgs a) {
  constexpr int V = kVec<T>, R = THREADS / TPR;
  __shared__ float lds[TPR == THREADS ? 2 * 7 * 16 : R * 64 * V];
  float w[NCH][V], cw[NCH][V], acc[1][NCH][V];
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    load_param<T, WHOLE>(a.w, a.wf32, chunk_col<T, TPR>(ch), a.D, 1.f, w[ch]);
    load_param<T, WHOLE>(a.cw, a.wf32, chunk_col<T, TPR>(ch), a.D, 0.f, cw[ch]);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[0][ch][j] = 0.f;
  }
  const float inv = 1.f / (float)a.D;
  const int64_t stride = (int64_t)gridDim.x * R;
  int64_t row = (int64_t)blockIdx.x * R + (int)threadIdx.x / TPR;
  Raw<T> nx[NCH], ndy[NCH], na[NCH];
  if (!a.a)
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int j = 0; j < V; ++j) na[ch].v[j] = (T)0.f;
  const auto fetch = [&](int64_t n) {
    load_row<T, TPR, NCH, WHOLE>(a.x, a.ldx, n, a, nx);
    load_row<T, TPR, NCH, WHOLE>(a.dy, a.lddy, n, a, ndy);
    if (a.a) load_row<T, TPR, NCH, WHOLE>(a.a, a.lda, n, a, na);
  };
  fetch(row);
  for (int turn = 0; row < a.N; row += stride, turn ^= 1) {
    const float r = a.rstd[row], mr = -a.mean[row] * r;
    Raw<T> x[NCH], dy[NCH], c[NCH];
    float s[7] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // past D: dy and a read 0 there, and so nothing of xh counts
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      x[ch] = nx[ch];
      dy[ch] = ndy[ch];
      c[ch] = na[ch];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (float)x[ch].v[j] * r + mr, d = (float)dy[ch].v[j], ca = (float)c[ch].v[j];
        const float g = d * w[ch][j], cd = d * cw[ch][j];
        s[0] += g;
        s[1] += g * xh;
        s[2] += ca;
        s[3] += ca * xh;
        s[4] += cd;
        s[5] += cd * xh;
        s[6] += ca * g;
      }
    }
    fetch(row + stride);
    row_sums<TPR, 7>(s, lds, turn);
    const float mg = s[0] * inv, mgx = s[1] * inv, ma = s[2] * inv, max_ = s[3] * inv;
    const float mt = s[4] * inv - r * (mgx * ma + max_ * mg);
    const float mtx = s[5] * inv - r * (2.f * mgx * max_);
    const float map = s[6] * inv - mg * ma - mgx * max_;
    // P(a) r = pa0 + r a + pa1 xh;  gx = o0 + o1 xh + o2 a + o3 g + r cw dy
    const float pa0 = -r * ma, pa1 = -r * max_;
    const float o0 = -r * mt, o1 = -(r * mtx + r * r * map), o2 = -r * r * mgx, o3 = -r * r * max_;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      float gdy[V], gx[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (float)x[ch].v[j] * r + mr, d = (float)dy[ch].v[j], ca = (float)c[ch].v[j];
        const float pa = ca * r + (xh * pa1 + pa0);
        acc[0][ch][j] += d * pa;
        gdy[j] = w[ch][j] * pa + cw[ch][j] * xh;
        gx[j] = (o0 + o1 * xh) + o2 * ca + d * (o3 * w[ch][j] + r * cw[ch][j]);
      }
      if (c0 >= a.D) break;
      if (a.gx) {
        if (a.cb) {
          float cb[V];
          load_param<T, WHOLE>(a.cb, a.wf32, c0, a.D, 0.f, cb);
#pragma unroll
          for (int j = 0; j < V; ++j) gdy[j] += cb[j];
        }
        store_chunk<T, WHOLE>((T*)a.gx + row * a.ldgx, c0, a.D, gdy);
      }
      if (a.y) store_chunk<T, WHOLE>((T*)a.y + row * a.ldy, c0, a.D, gx);
    }
  }
  if (a.part) store_sums<T, TPR, NCH, THREADS, WHOLE, 1>(a, acc, lds);
}

// out_k[col] = sum over groups of part[group][k][col], in group order within
// each of 64 lanes' strides, the strides in lane order.
template <typename TP>
__global__ __launch_bounds__(1024) void k_norm_sums(const float* part, int groups, int nsum, int D, void* o0,
                                                    void* o1) {
  __shared__ float lds[64][17];
  const int c = threadIdx.x & 15, s = threadIdx.x >> 4, k = blockIdx.y;
  const int col = blockIdx.x * 16 + c;
  float t = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int g = s; g < groups; g += 64) t += part[((int64_t)g * nsum + k) * D + col];
  }
  lds[s][c] = t;
  __syncthreads();
  if (s == 0 && col < D) {
    float v = 0.f;
#pragma unroll 16
    for (int i = 0; i < 64; ++i) v += lds[i][c];
    TP* o = (TP*)(k == 0 ? o0 : o1);
    if (o) o[col] = (TP)v;
  }
}

struct Shape {
  int tpr, nch, threads;  // threads of a row, chunks of each, threads of a workgroup
  int per() const { return threads / tpr; }
};

// One chunk a thread as long as a workgroup can hold the row that way: the
// fewest registers, so the most rows in flight (backward of 65536 x 4096 bf16:
// 453 us with 256 threads of two chunks, 313 with 512 of one).  A row in more
// than one wave is a workgroup's: its barriers must be met by all.
template <typename T>
Shape norm_shape(int64_t D) {
  const int64_t c = (D + kVec<T> - 1) / kVec<T>;  // chunks of a row
  if (c <= 64) return {64, 1, 256};
  if (c <= 128) return {128, 1, 128};
  if (c <= 256) return {256, 1, 256};
  if (c <= 512) return {512, 1, 512};
  if (c <= 1024) return {1024, 1, 1024};
  if (c <= 2048) return {1024, 2, 1024};
  return {1024, 4, 1024};
}

#define NORM_SHAPES(KERNEL, T, WHOLE, sh, grid, st, args)                                                \
  do {                                                                                                   \
    if (sh.tpr == 64) KERNEL<T, 64, 1, 256, WHOLE><<<grid, 256, 0, st>>>(args);                          \
    else if (sh.tpr == 128) KERNEL<T, 128, 1, 128, WHOLE><<<grid, 128, 0, st>>>(args);                   \
    else if (sh.tpr == 256) KERNEL<T, 256, 1, 256, WHOLE><<<grid, 256, 0, st>>>(args);                   \
    else if (sh.tpr == 512) KERNEL<T, 512, 1, 512, WHOLE><<<grid, 512, 0, st>>>(args);                   \
    else if (sh.nch == 1) KERNEL<T, 1024, 1, 1024, WHOLE><<<grid, 1024, 0, st>>>(args);                  \
    else if (sh.nch == 2) KERNEL<T, 1024, 2, 1024, WHOLE><<<grid, 1024, 0, st>>>(args);                  \
    else KERNEL<T, 1024, 4, 1024, WHOLE><<<grid, 1024, 0, st>>>(args);                                   \
  } while (0)
#define NORM_DISPATCH(KERNEL, T, sh, grid, st, args)                          \
  do {                                                                        \
    if (args.D % kVec<T> == 0) NORM_SHAPES(KERNEL, T, true, sh, grid, st, args); \
    else NORM_SHAPES(KERNEL, T, false, sh, grid, st, args);                   \
  } while (0)

#define NORM_TYPES(dtype, ...)                                     \
  do {                                                             \
    if ((dtype) == TTT_F16) { typedef _Float16 T; __VA_ARGS__; }   \
    else if ((dtype) == TTT_BF16) { typedef __bf16 T; __VA_ARGS__; } \
    else { typedef float T; __VA_ARGS__; }                         \
  } while (0)

// Workgroups of a launch at most, in threads: eight of 256 per CU; half as
// many where column sums are formed, each of which is written and read once;
// and a quarter where that leaves a workgroup fewer than 16 rows, so that the
// sums are fewer bytes beside the rows (with half and with a quarter, backward
// and its sums: 2999 x 1003 fp16 20.6 and 18.3 us, 8192 x 384 fp32 15.9 and
// 15.2; gg of 8192 x 2048 bf16 45.4 and 41.2; backward of 65536 x 4096 bf16 303
// and 419).
constexpr int64_t kFwdThreads = 2048 * 256, kSumThreads = 1024 * 256;

int walkers(const ttt_norm_problem* p, const Shape& sh, int64_t threads) {
  const int64_t n = (p->rows + sh.per() - 1) / sh.per(), most = threads / sh.threads;
  return (int)(n < most ? n : most);
}
int groups_of(const ttt_norm_problem* p, const Shape& sh) {
  const int n = walkers(p, sh, kSumThreads);
  return p->rows < 16ll * sh.per() * n ? walkers(p, sh, kSumThreads / 2) : n;
}

Shape shape_of(const ttt_norm_problem* p) {
  return p->dtype == TTT_F32 ? norm_shape<float>(p->cols) : norm_shape<_Float16>(p->cols);
}

int check(const ttt_norm_problem* p) {
  if (!p) return ops_fail(TTT_ERR_INVALID_ARGUMENT, "layer norm: null problem");
  if (p->dtype != TTT_F16 && p->dtype != TTT_BF16 && p->dtype != TTT_F32)
    return ops_fail(TTT_ERR_UNSUPPORTED, "layer norm: dtype code %d is not f16/bf16/f32", p->dtype);
  if (p->param_dtype != p->dtype && p->param_dtype != TTT_F32)
    return ops_fail(TTT_ERR_UNSUPPORTED, "layer norm: parameters of dtype code %d: that of x, or f32", p->param_dtype);
  if (p->rows < 1 || p->rows > 0x7fffffff)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "layer norm: rows %lld: must be 1 .. 2^31 - 1", (long long)p->rows);
  const int64_t most = p->dtype == TTT_F32 ? 16384 : 32768;
  if (p->cols < 1 || p->cols > most)
    return ops_fail(TTT_ERR_UNSUPPORTED, "layer norm: rows of %lld values: 1 .. %lld for this type",
                    (long long)p->cols, (long long)most);
  return TTT_OK;
}

int take(const ttt_norm_problem* p, const ttt_rows* r, const char* name, bool need, const void** ptr, int64_t* ld) {
  *ptr = r ? r->data : nullptr;
  *ld = r ? r->stride : 0;
  if (!*ptr) return need ? ops_fail(TTT_ERR_INVALID_ARGUMENT, "layer norm: %s: null pointer", name) : TTT_OK;
  if (*ld < p->cols)
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "layer norm: %s: row stride %lld below the row length %lld", name,
                    (long long)*ld, (long long)p->cols);
  if ((uintptr_t)*ptr % (p->dtype == TTT_F32 ? 4 : 2))
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "layer norm: %s: base pointer not aligned to its type", name);
  return TTT_OK;
}

#define TRY(x)                     \
  do {                             \
    const int rc_ = (x);           \
    if (rc_ != TTT_OK) return rc_; \
  } while (0)

int finish(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return ops_fail(TTT_ERR_LAUNCH, "%s: launch failed: %s", what, hipGetErrorString(e));
  return TTT_OK;
}

void launch_sums(const ttt_norm_problem* p, const float* part, int groups, int nsum, void* o0, void* o1,
                 hipStream_t st) {
  const dim3 grid((unsigned)((p->cols + 15) / 16), nsum);
  NORM_TYPES(p->param_dtype, (k_norm_sums<T><<<grid, 1024, 0, st>>>(part, groups, nsum, (int)p->cols, o0, o1)));
}

}  // namespace
}  // namespace ttt

using namespace ttt;

extern "C" {

int64_t ttt_norm_workspace_size(const ttt_norm_problem* p) {
  if (check(p) != TTT_OK) return -1;
  return (int64_t)groups_of(p, shape_of(p)) * 2 * p->cols * (int64_t)sizeof(float);
}

int ttt_norm_fwd(const ttt_norm_problem* p, const ttt_rows* x, const void* weight, const void* bias,
                 const ttt_rows* y, float* mean, float* rstd, void* stream) {
  TRY(check(p));
  NormArgs a;
  memset(&a, 0, sizeof(a));
  const void* yp;
  TRY(take(p, x, "x", true, &a.x, &a.ldx));
  TRY(take(p, y, "y", true, &yp, &a.ldy));
  if ((mean == nullptr) != (rstd == nullptr))
    return ops_fail(TTT_ERR_INVALID_ARGUMENT, "layer norm: mean and rstd: both or neither");
  a.y = const_cast<void*>(yp);
  a.w = weight;
  a.b = bias;
  a.mean = mean;
  a.rstd = rstd;
  a.N = (int)p->rows;
  a.D = (int)p->cols;
  a.wf32 = p->param_dtype == TTT_F32;
  a.eps = p->eps;
  const Shape sh = shape_of(p);
  const unsigned grid = (unsigned)walkers(p, sh, kFwdThreads);
  const hipStream_t st = (hipStream_t)stream;
  NORM_TYPES(p->dtype, NORM_DISPATCH(k_norm_fwd, T, sh, grid, st, a));
  return finish("ttt_norm_fwd");
}

int ttt_norm_bwd(const ttt_norm_problem* p, const ttt_rows* x, const void* weight, const ttt_rows* dy,
                 const float* mean, const float* rstd, const ttt_rows* dx, void* dweight, void* dbias,
                 void* workspace, int64_t workspace_bytes, void* stream) {
  TRY(check(p));
  NormArgs a;
  memset(&a, 0, sizeof(a));
  const void* dxp;
  TRY(take(p, x, "x", true, &a.x, &a.ldx));
  TRY(take(p, dy, "dy", true, &a.dy, &a.lddy));
  TRY(take(p, dx, "dx", false, &dxp, &a.ldy));
  if (!mean || !rstd) return ops_fail(TTT_ERR_INVALID_ARGUMENT, "layer norm: mean and rstd are needed");
  const bool sums = dweight || dbias;
  if (!dxp && !sums) return TTT_OK;
  if (sums && (!workspace || workspace_bytes < ttt_norm_workspace_size(p)))
    return ops_fail(TTT_ERR_WORKSPACE, "ttt_norm_bwd: workspace of %lld bytes, needs %lld",
                    workspace ? (long long)workspace_bytes : 0ll, (long long)ttt_norm_workspace_size(p));
  a.y = const_cast<void*>(dxp);
  a.w = weight;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.part = sums ? (float*)workspace : nullptr;
  a.N = (int)p->rows;
  a.D = (int)p->cols;
  a.wf32 = p->param_dtype == TTT_F32;
  const Shape sh = shape_of(p);
  const int groups = groups_of(p, sh);
  const hipStream_t st = (hipStream_t)stream;
  NORM_TYPES(p->dtype, NORM_DISPATCH(k_norm_bwd, T, sh, groups, st, a));
  if (sums) launch_sums(p, a.part, groups, 2, dweight, dbias, st);
  return finish("ttt_norm_bwd");
}

int ttt_norm_gg(const ttt_norm_problem* p, const ttt_rows* x, const void* weight, const ttt_rows* dy,
                const float* mean, const float* rstd, const ttt_rows* ca, const void* cw, const void* cb,
                const ttt_rows* gx, void* gw, const ttt_rows* gdy, void* workspace, int64_t workspace_bytes,
                void* stream) {
  TRY(check(p));
  NormArgs a;
  memset(&a, 0, sizeof(a));
  const void *gxp, *gdyp;
  TRY(take(p, x, "x", true, &a.x, &a.ldx));
  TRY(take(p, dy, "dy", true, &a.dy, &a.lddy));
  TRY(take(p, ca, "a", false, &a.a, &a.lda));
  TRY(take(p, gx, "gx", false, &gxp, &a.ldy));
  TRY(take(p, gdy, "gdy", false, &gdyp, &a.ldgx));
  if (!mean || !rstd) return ops_fail(TTT_ERR_INVALID_ARGUMENT, "layer norm: mean and rstd are needed");
  if (!gxp && !gdyp && !gw) return TTT_OK;
  if (gw && (!workspace || workspace_bytes < ttt_norm_workspace_size(p)))
    return ops_fail(TTT_ERR_WORKSPACE, "ttt_norm_gg: workspace of %lld bytes, needs %lld",
                    workspace ? (long long)workspace_bytes : 0ll, (long long)ttt_norm_workspace_size(p));
  a.y = const_cast<void*>(gxp);
  a.gx = const_cast<void*>(gdyp);
  a.w = weight;
  a.cw = cw;
  a.cb = cb;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.part = gw ? (float*)workspace : nullptr;
  a.N = (int)p->rows;
  a.D = (int)p->cols;
  a.wf32 = p->param_dtype == TTT_F32;
  const Shape sh = shape_of(p);
  const int groups = groups_of(p, sh);
  const hipStream_t st = (hipStream_t)stream;
  NORM_TYPES(p->dtype, NORM_DISPATCH(k_norm_gg, T, sh, groups, st, a));
  if (gw) launch_sums(p, a.part, groups, 1, gw, nullptr, st);
  return finish("ttt_norm_gg");
}

}  // extern "C"

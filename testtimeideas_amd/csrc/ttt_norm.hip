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

// Eight (four) consecutive values at p as fp32; the loads are 16 bytes wide
// whatever p's alignment is (global memory takes any).  Values past D read 0.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int col, int D, float* v) {
  constexpr int V = kVec<T>;
  T r[V];
  if (col + V <= D) {
    __builtin_memcpy(r, row + col, 16);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)r[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = col + j < D ? (float)row[col + j] : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* row, int col, int D, const float* v) {
  constexpr int V = kVec<T>;
  if (col + V <= D) {
    T r[V];
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = (T)v[j];
    __builtin_memcpy(row + col, r, 16);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (col + j < D) row[col + j] = (T)v[j];
  }
}

// V parameters at column col: of type T, or fp32 (f32); `none` where p is null.
template <typename T>
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
    load_chunk<T>((const T*)p, col, D, v);
  }
}

__device__ __forceinline__ float lane_swap_sum(float x, int mask) {
  return x + __shfl_xor(x, mask);
}

// Sums of NS values over the threads of a row (TPR = 64: a wave; more: the
// workgroup, through LDS), to every thread.
template <int TPR, int NS>
__device__ __forceinline__ void row_sums(float* s, float* lds) {
#pragma unroll
  for (int k = 0; k < NS; ++k)
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) s[k] = lane_swap_sum(s[k], m);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int w = threadIdx.x >> 6;
    __syncthreads();  // the sums of the call before have been read
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

// Thread's chunk `ch` of a row: columns of chunk-major order, so a wave's
// loads of one chunk are contiguous.
template <typename T, int TPR>
__device__ __forceinline__ int chunk_col(int ch) {
  return (ch * TPR + (int)(threadIdx.x % TPR)) * kVec<T>;
}

template <typename T, int TPR, int NCH, int THREADS>
__global__ __launch_bounds__(THREADS) void k_norm_fwd(NormArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float lds[2 * 16];
  const int row = blockIdx.x * (THREADS / TPR) + (int)threadIdx.x / TPR;
  if (TPR == 64 && row >= a.N) return;
  const T* x = (const T*)a.x + (int64_t)row * a.ldx;
  T* y = (T*)a.y + (int64_t)row * a.ldy;
  float v[NCH][V];
  float s[1] = {0.f};
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    load_chunk<T>(x, chunk_col<T, TPR>(ch), a.D, v[ch]);
#pragma unroll
    for (int j = 0; j < V; ++j) s[0] += v[ch][j];
  }
  row_sums<TPR, 1>(s, lds);
  const float inv = 1.f / (float)a.D, mu = s[0] * inv;
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
  row_sums<TPR, 1>(q, lds);
  const float r = 1.f / sqrtf(q[0] * inv + a.eps);
  if (a.mean && threadIdx.x % TPR == 0) {
    a.mean[row] = mu;
    a.rstd[row] = r;
  }
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    const int c0 = chunk_col<T, TPR>(ch);
    if (c0 >= a.D) break;
    float w[V], b[V];
    load_param<T>(a.w, a.wf32, c0, a.D, 1.f, w);
    load_param<T>(a.b, a.wf32, c0, a.D, 0.f, b);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = v[ch][j] * r * w[j] + b[j];
    store_chunk<T>(y, c0, a.D, w);
  }
}

// The column sums of a workgroup's rows to part[group][k][D].  With TPR = 64
// the waves hold sums of the same columns: added through LDS in wave order.
template <typename T, int TPR, int NCH, int THREADS, int NSUM>
__device__ __forceinline__ void store_sums(const NormArgs& a, float (*acc)[NCH][kVec<T>], float* lds) {
  constexpr int V = kVec<T>, W = THREADS / TPR, COLS = 64 * V;
  float* part = a.part + (int64_t)blockIdx.x * NSUM * a.D;
#pragma unroll
  for (int k = 0; k < NSUM; ++k)
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      if constexpr (TPR == THREADS) {
        store_chunk<float>(part + (int64_t)k * a.D, c0, a.D, acc[k][ch]);
        if constexpr (V == 8) store_chunk<float>(part + (int64_t)k * a.D, c0 + 4, a.D, acc[k][ch] + 4);
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

template <typename T, int TPR, int NCH, int THREADS>
__global__ __launch_bounds__(THREADS) void k_norm_bwd(NormArgs a) {
  constexpr int V = kVec<T>, R = THREADS / TPR;
  __shared__ float lds[TPR == THREADS ? 64 : R * 64 * V];
  float w[NCH][V], acc[2][NCH][V];
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    load_param<T>(a.w, a.wf32, chunk_col<T, TPR>(ch), a.D, 1.f, w[ch]);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[0][ch][j] = acc[1][ch][j] = 0.f;
  }
  const float inv = 1.f / (float)a.D;
  for (int row = blockIdx.x * R + (int)threadIdx.x / TPR; row < a.N; row += gridDim.x * R) {
    const T* x = (const T*)a.x + (int64_t)row * a.ldx;
    const T* dy = (const T*)a.dy + (int64_t)row * a.lddy;
    const float mu = a.mean[row], r = a.rstd[row];
    float xh[NCH][V], g[NCH][V], s[2] = {0.f, 0.f};
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      load_chunk<T>(x, c0, a.D, xh[ch]);
      load_chunk<T>(dy, c0, a.D, g[ch]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[ch][j] = (xh[ch][j] - mu) * r;  // past D: dy reads 0 there
        acc[0][ch][j] += g[ch][j] * xh[ch][j];
        acc[1][ch][j] += g[ch][j];
        g[ch][j] *= w[ch][j];
        s[0] += g[ch][j];
        s[1] += g[ch][j] * xh[ch][j];
      }
    }
    if (!a.y) continue;
    row_sums<TPR, 2>(s, lds);
    const float m1 = s[0] * inv, m2 = s[1] * inv;
    T* dx = (T*)a.y + (int64_t)row * a.ldy;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      if (c0 >= a.D) break;
#pragma unroll
      for (int j = 0; j < V; ++j) g[ch][j] = r * (g[ch][j] - m1 - xh[ch][j] * m2);
      store_chunk<T>(dx, c0, a.D, g[ch]);
    }
  }
  if (a.part) store_sums<T, TPR, NCH, THREADS, 2>(a, acc, lds);
}

template <typename T, int TPR, int NCH, int THREADS>
__global__ __launch_bounds__(THREADS) void k_norm_gg(NormArgs a) {
  constexpr int V = kVec<T>, R = THREADS / TPR;
  __shared__ float lds[TPR == THREADS ? 64 : R * 64 * V];
  float w[NCH][V], acc[1][NCH][V];
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch) {
    load_param<T>(a.w, a.wf32, chunk_col<T, TPR>(ch), a.D, 1.f, w[ch]);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[0][ch][j] = 0.f;
  }
  const float inv = 1.f / (float)a.D;
  for (int row = blockIdx.x * R + (int)threadIdx.x / TPR; row < a.N; row += gridDim.x * R) {
    const T* x = (const T*)a.x + (int64_t)row * a.ldx;
    const T* dyp = (const T*)a.dy + (int64_t)row * a.lddy;
    const float mu = a.mean[row], r = a.rstd[row];
    float xh[NCH][V], dy[NCH][V], c[NCH][V], s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      load_chunk<T>(x, c0, a.D, xh[ch]);
      load_chunk<T>(dyp, c0, a.D, dy[ch]);
      if (a.a) {
        load_chunk<T>((const T*)a.a + (int64_t)row * a.lda, c0, a.D, c[ch]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) c[ch][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[ch][j] = c0 + j < a.D ? (xh[ch][j] - mu) * r : 0.f;
        const float g = dy[ch][j] * w[ch][j];
        s[0] += g;
        s[1] += g * xh[ch][j];
        s[2] += c[ch][j];
        s[3] += c[ch][j] * xh[ch][j];
      }
    }
    row_sums<TPR, 4>(s, lds);
    const float mg = s[0] * inv, mgx = s[1] * inv, ma = s[2] * inv, max_ = s[3] * inv;
    // second round: mean(t), mean(t xh), mean(a P(g)); gdy goes out on the way
    float u[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      float cw[V], cb[V], gdy[V];
      load_param<T>(a.cw, a.wf32, c0, a.D, 0.f, cw);
      load_param<T>(a.cb, a.wf32, c0, a.D, 0.f, cb);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool in = c0 + j < a.D;
        const float g = dy[ch][j] * w[ch][j];
        const float ca = c[ch][j];
        const float pa = in ? ca - ma - xh[ch][j] * max_ : 0.f;
        const float pg = g - mg - xh[ch][j] * mgx;
        acc[0][ch][j] += dy[ch][j] * r * pa;
        gdy[j] = w[ch][j] * r * pa + cw[j] * xh[ch][j] + cb[j];
        const float t = cw[j] * dy[ch][j] - r * (ca * mgx + g * max_);
        c[ch][j] = t;
        u[0] += t;
        u[1] += t * xh[ch][j];
        u[2] += in ? (ca - ma) * pg : 0.f;  // mean(pg) is 0: a without its own mean
      }
      if (a.gx && c0 < a.D) store_chunk<T>((T*)a.gx + (int64_t)row * a.ldgx, c0, a.D, gdy);
    }
    if (!a.y) continue;
    row_sums<TPR, 3>(u, lds);
    const float mt = u[0] * inv, mtx = r * (u[1] * inv) + r * r * (u[2] * inv);
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int c0 = chunk_col<T, TPR>(ch);
      if (c0 >= a.D) break;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = r * (c[ch][j] - mt) - xh[ch][j] * mtx;
      store_chunk<T>((T*)a.y + (int64_t)row * a.ldy, c0, a.D, o);
    }
  }
  if (a.part) store_sums<T, TPR, NCH, THREADS, 1>(a, acc, lds);
}

// out_k[col] = sum over groups of part[group][k][col], in group order within
// each of 32 lanes' strides, the strides in lane order.
template <typename TP>
__global__ __launch_bounds__(1024) void k_norm_sums(const float* part, int groups, int nsum, int D, void* o0,
                                                    void* o1) {
  __shared__ float lds[32][33];
  const int c = threadIdx.x & 31, s = threadIdx.x >> 5, k = blockIdx.y;
  const int col = blockIdx.x * 32 + c;
  float t = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int g = s; g < groups; g += 32) t += part[((int64_t)g * nsum + k) * D + col];
  }
  lds[s][c] = t;
  __syncthreads();
  if (s == 0 && col < D) {
    float v = 0.f;
    for (int i = 0; i < 32; ++i) v += lds[i][c];
    TP* o = (TP*)(k == 0 ? o0 : o1);
    if (o) o[col] = (TP)v;
  }
}

// Rows walked by one workgroup at least, where column sums are formed: their
// partial sums are [groups][2][D] fp32, written and read once.
constexpr int kNormGroups = 1024;

struct Shape {
  int tpr, nch, threads;
};

// The narrowest row layout that holds D values in registers.
template <typename T>
Shape norm_shape(int64_t D) {
  const int64_t c = (D + kVec<T> - 1) / kVec<T>;  // chunks of a row
  if (c <= 64) return {64, 1, 256};
  if (c <= 128) return {64, 2, 256};
  if (c <= 256) return {256, 1, 256};
  if (c <= 512) return {256, 2, 256};
  if (c <= 1024) return {1024, 1, 1024};
  if (c <= 2048) return {1024, 2, 1024};
  return {1024, 4, 1024};
}

#define NORM_DISPATCH(KERNEL, T, sh, grid, st, args)                                                  \
  do {                                                                                                \
    if (sh.tpr == 64 && sh.nch == 1) KERNEL<T, 64, 1, 256><<<grid, 256, 0, st>>>(args);               \
    else if (sh.tpr == 64) KERNEL<T, 64, 2, 256><<<grid, 256, 0, st>>>(args);                         \
    else if (sh.tpr == 256 && sh.nch == 1) KERNEL<T, 256, 1, 256><<<grid, 256, 0, st>>>(args);        \
    else if (sh.tpr == 256) KERNEL<T, 256, 2, 256><<<grid, 256, 0, st>>>(args);                       \
    else if (sh.nch == 1) KERNEL<T, 1024, 1, 1024><<<grid, 1024, 0, st>>>(args);                      \
    else if (sh.nch == 2) KERNEL<T, 1024, 2, 1024><<<grid, 1024, 0, st>>>(args);                      \
    else KERNEL<T, 1024, 4, 1024><<<grid, 1024, 0, st>>>(args);                                       \
  } while (0)

#define NORM_TYPES(dtype, ...)                                     \
  do {                                                             \
    if ((dtype) == TTT_F16) { typedef _Float16 T; __VA_ARGS__; }   \
    else if ((dtype) == TTT_BF16) { typedef __bf16 T; __VA_ARGS__; } \
    else { typedef float T; __VA_ARGS__; }                         \
  } while (0)

int groups_of(const ttt_norm_problem* p, const Shape& sh) {
  const int64_t per = sh.threads / sh.tpr, n = (p->rows + per - 1) / per;
  return (int)(n < kNormGroups ? n : kNormGroups);
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
  const dim3 grid((unsigned)((p->cols + 31) / 32), nsum);
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
  const int per = sh.threads / sh.tpr;
  const unsigned grid = (unsigned)((p->rows + per - 1) / per);
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

// rtg_layernorm.hip — layer norm forward and backward over the last axis (rows) or over the channel axis of feature maps
// (see include/rtg.h, rtg_layernorm_*).
//
//   y = (x - mean) * rstd * w + b                                    per row: mean, var over n elements
//   g = dy * w;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat));  dw = sum dy * xhat;  db = sum dy
//
// ~8 (forward) and ~16 (backward) operations per element of 4 .. 12 bytes moved: bound by HBM.
#include "rtg_vec.h"

namespace {

constexpr int LOOP_THREADS = 256;
constexpr int FIN_COLS = 32, FIN_ROWS = 32;

struct LnShape {
  long long outer, n, inner, xo, xn;      // x[o * xo + c * xn + t]; everything else contiguous
  float nf, eps;                          // n as a float (sums are divided by it: the mean of equal values is that value)
  int pbf;                                // weight / bias (and their gradients) are bf16
};

__device__ __forceinline__ float param_at(const void* p, int bf, long long i, float dflt) {
  if (!p) return dflt;
  return bf ? rtg_up(reinterpret_cast<const rtg_bf16*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}

// ---------------------------------------------------------------------------------------------------------------------
// Kernels for any size.  A row that no register kernel holds is read once per sum; the later reads come from L2.
// ---------------------------------------------------------------------------------------------------------------------
template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_row_loop_fwd(LnShape s, const T* __restrict__ x, const void* __restrict__ w,
                                                                const void* __restrict__ b, T* __restrict__ y,
                                                                float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float red[4];
  for (long long row = blockIdx.x; row < s.outer; row += gridDim.x) {
    const T* xr = x + row * s.xo;
    float acc = 0.f;
    for (long long i = threadIdx.x; i < s.n; i += LOOP_THREADS) acc += rtg_up(xr[i]);
    const float mean = rtg_block_sum(acc, red) / s.nf;
    acc = 0.f;
    for (long long i = threadIdx.x; i < s.n; i += LOOP_THREADS) {
      const float d = rtg_up(xr[i]) - mean;
      acc += d * d;
    }
    const float rstd = 1.f / sqrtf(rtg_block_sum(acc, red) / s.nf + s.eps);
    for (long long i = threadIdx.x; i < s.n; i += LOOP_THREADS)
      rtg_down((rtg_up(xr[i]) - mean) * rstd * param_at(w, s.pbf, i, 1.f) + param_at(b, s.pbf, i, 0.f), y[row * s.n + i]);
    if (mean_out && threadIdx.x == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_row_loop_dx(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                               const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                               const void* __restrict__ w, T* __restrict__ dx) {
  __shared__ float red[4];
  for (long long row = blockIdx.x; row < s.outer; row += gridDim.x) {
    const T *xr = x + row * s.xo, *gr = dy + row * s.n;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float a1 = 0.f, a2 = 0.f;
    for (long long i = threadIdx.x; i < s.n; i += LOOP_THREADS) {
      const float g = rtg_up(gr[i]) * param_at(w, s.pbf, i, 1.f);
      a1 += g;
      a2 += g * ((rtg_up(xr[i]) - mean) * rstd);
    }
    const float c1 = rtg_block_sum(a1, red) / s.nf, c2 = rtg_block_sum(a2, red) / s.nf;
    for (long long i = threadIdx.x; i < s.n; i += LOOP_THREADS) {
      const float g = rtg_up(gr[i]) * param_at(w, s.pbf, i, 1.f);
      rtg_down(rstd * (g - c1 - (rtg_up(xr[i]) - mean) * rstd * c2), dx[row * s.n + i]);
    }
  }
}

// partial dw, db of slice blockIdx.y of the rows: 64 adjacent columns a block, its four waves every fourth row
template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_row_loop_dw(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd,
                                                               float* __restrict__ part, int slices) {
  __shared__ float red[2][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long i = (long long)blockIdx.x * 64 + lane;
  float aw = 0.f, ab = 0.f;
  if (i < s.n)
    for (long long row = blockIdx.y * 4 + wave; row < s.outer; row += 4 * slices) {
      const float g = rtg_up(dy[row * s.n + i]);
      aw += g * ((rtg_up(x[row * s.xo + i]) - mean[row]) * rstd[row]);
      ab += g;
    }
  red[0][wave][lane] = aw;
  red[1][wave][lane] = ab;
  __syncthreads();
  if (wave < 2 && i < s.n)
    part[((long long)blockIdx.y * 2 + wave) * s.n + i] =
        (red[wave][0][lane] + red[wave][1][lane]) + (red[wave][2][lane] + red[wave][3][lane]);
}

// the sum over a block's four waves of `v` at each lane, in every wave
__device__ __forceinline__ float wave_column_sum(float v, float (&red)[4][64]) {
  const int lane = threadIdx.x & 63;
  __syncthreads();
  red[threadIdx.x >> 6][lane] = v;
  __syncthreads();
  return (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

// feature maps: a lane is a position, the four waves share the channels
template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_map_loop_fwd(LnShape s, const T* __restrict__ x, const void* __restrict__ w,
                                                                const void* __restrict__ b, T* __restrict__ y,
                                                                float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long tiles = (s.inner + 63) / 64;
  for (long long tile = blockIdx.x; tile < s.outer * tiles; tile += gridDim.x) {
    const long long o = tile / tiles, t = (tile - o * tiles) * 64 + lane;
    const bool in = t < s.inner;
    const T* xp = x + o * s.xo + t;
    float acc = 0.f;
    if (in)
      for (long long c = wave; c < s.n; c += 4) acc += rtg_up(xp[c * s.xn]);
    const float mean = wave_column_sum(acc, red) / s.nf;
    acc = 0.f;
    if (in)
      for (long long c = wave; c < s.n; c += 4) {
        const float d = rtg_up(xp[c * s.xn]) - mean;
        acc += d * d;
      }
    const float rstd = 1.f / sqrtf(wave_column_sum(acc, red) / s.nf + s.eps);
    if (!in) continue;
    T* yp = y + o * s.n * s.inner + t;
    for (long long c = wave; c < s.n; c += 4)
      rtg_down((rtg_up(xp[c * s.xn]) - mean) * rstd * param_at(w, s.pbf, c, 1.f) + param_at(b, s.pbf, c, 0.f), yp[c * s.inner]);
    if (mean_out && wave == 0) {
      mean_out[o * s.inner + t] = mean;
      rstd_out[o * s.inner + t] = rstd;
    }
  }
}

template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_map_loop_dx(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                               const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                               const void* __restrict__ w, T* __restrict__ dx) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long tiles = (s.inner + 63) / 64;
  for (long long tile = blockIdx.x; tile < s.outer * tiles; tile += gridDim.x) {
    const long long o = tile / tiles, t = (tile - o * tiles) * 64 + lane;
    const bool in = t < s.inner;
    const T *xp = x + o * s.xo + t, *gp = dy + o * s.n * s.inner + t;
    float mean = 0.f, rstd = 0.f, a1 = 0.f, a2 = 0.f;
    if (in) {
      mean = mean_in[o * s.inner + t];
      rstd = rstd_in[o * s.inner + t];
      for (long long c = wave; c < s.n; c += 4) {
        const float g = rtg_up(gp[c * s.inner]) * param_at(w, s.pbf, c, 1.f);
        a1 += g;
        a2 += g * ((rtg_up(xp[c * s.xn]) - mean) * rstd);
      }
    }
    const float c1 = wave_column_sum(a1, red) / s.nf, c2 = wave_column_sum(a2, red) / s.nf;
    if (!in) continue;
    T* dp = dx + o * s.n * s.inner + t;
    for (long long c = wave; c < s.n; c += 4) {
      const float g = rtg_up(gp[c * s.inner]) * param_at(w, s.pbf, c, 1.f);
      rtg_down(rstd * (g - c1 - (rtg_up(xp[c * s.xn]) - mean) * rstd * c2), dp[c * s.inner]);
    }
  }
}

// partial dw, db of one channel (blockIdx.x) over slice blockIdx.y of the positions of all clips
template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_map_loop_dw(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd,
                                                               float* __restrict__ part, int slices) {
  __shared__ float red[4];
  const long long total = s.outer * s.inner;
  for (long long c = blockIdx.x; c < s.n; c += gridDim.x) {
    float aw = 0.f, ab = 0.f;
    for (long long p = (long long)blockIdx.y * LOOP_THREADS + threadIdx.x; p < total; p += (long long)slices * LOOP_THREADS) {
      const long long o = p / s.inner, t = p - o * s.inner;
      const float g = rtg_up(dy[(o * s.n + c) * s.inner + t]);
      aw += g * ((rtg_up(x[o * s.xo + c * s.xn + t]) - mean[p]) * rstd[p]);
      ab += g;
    }
    aw = rtg_block_sum(aw, red);
    ab = rtg_block_sum(ab, red);
    if (threadIdx.x == 0) {
      part[((long long)blockIdx.y * 2) * s.n + c] = aw;
      part[((long long)blockIdx.y * 2 + 1) * s.n + c] = ab;
    }
  }
}

// dw, db = the sums of their `slices` partials [slice][dw | db][n], each in the order of the slices: 32 columns a block, a
// column's slices over 32 threads (so that the reads of a column are in flight together), then a fixed tree
__global__ __launch_bounds__(FIN_COLS* FIN_ROWS) void ln_finish(const float* __restrict__ part, int slices, long long n,
                                                                void* __restrict__ dw, void* __restrict__ db, int pbf) {
  __shared__ float red[FIN_ROWS][FIN_COLS + 1];
  void* const out = blockIdx.y ? db : dw;
  if (!out) return;
  const int col = threadIdx.x % FIN_COLS, r = threadIdx.x / FIN_COLS;
  const long long i = (long long)blockIdx.x * FIN_COLS + col;
  float acc = 0.f;
  if (i < n)
    for (int q = r; q < slices; q += FIN_ROWS) acc += part[((long long)q * 2 + blockIdx.y) * n + i];
  red[r][col] = acc;
  __syncthreads();
#pragma unroll
  for (int h = FIN_ROWS / 2; h > 0; h >>= 1) {
    if (r < h) red[r][col] += red[r + h][col];
    __syncthreads();
  }
  if (r == 0 && i < n) {
    if (pbf) rtg_down(red[0][col], reinterpret_cast<rtg_bf16*>(out)[i]);
    else reinterpret_cast<float*>(out)[i] = red[0][col];
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
inline long long lmin(long long a, long long b) { return a < b ? a : b; }

int check_desc(const RtgLayerNormDesc* d) {
  if (!d) return RTG_ENULL;
  if (d->n < 1 || d->outer < 0 || d->inner < 0 || d->x_outer < 0 || d->x_n < 0 || !(d->eps >= 0.f)) return RTG_EINVAL;
  if (d->inner == 1 && d->n > 1 && d->x_n != 1) return RTG_EINVAL;
  long long t;
  if (__builtin_mul_overflow(d->outer, d->n, &t) || __builtin_mul_overflow(t, d->inner, &t) || t > (1ll << 60)) return RTG_ERANGE;
  if (__builtin_mul_overflow(d->outer, d->x_outer, &t) || t > (1ll << 60)) return RTG_ERANGE;
  if (__builtin_mul_overflow(d->n, d->x_n, &t) || t > (1ll << 60) || d->n > 0x7fffffffll) return RTG_ERANGE;
  return RTG_OK;
}

LnShape shape_of(const RtgLayerNormDesc* d) {
  return LnShape{d->outer, d->n, d->inner, d->x_outer, d->x_n, (float)d->n, d->eps, d->param_bf16 != 0};
}

bool is_rows(const RtgLayerNormDesc* d) { return d->inner == 1; }

// slices the sums over rows / positions are cut into: enough blocks for the chip, few partials beside what they sum
int dw_slices(const RtgLayerNormDesc* d) {
  const long long cols = is_rows(d) ? (d->n + 63) / 64 : d->n;
  const long long work = is_rows(d) ? (d->outer + 15) / 16 : (d->outer * d->inner + 1023) / 1024;
  long long s = lmin(work, (2048 + cols - 1) / cols);
  return (int)(s < 1 ? 1 : lmin(s, 1024));
}

template <class T>
int forward(const RtgLayerNormDesc* d, const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, hipStream_t st) {
  const LnShape s = shape_of(d);
  const T* xt = reinterpret_cast<const T*>(x);
  T* yt = reinterpret_cast<T*>(y);
  if (is_rows(d)) {
    RTG_KLAUNCH(ln_row_loop_fwd<T>, dim3((unsigned)lmin(d->outer, 1 << 20)), dim3(LOOP_THREADS), 0, st, s, xt, w, b, yt, mean, rstd);
  } else {
    const long long tiles = d->outer * ((d->inner + 63) / 64);
    RTG_KLAUNCH(ln_map_loop_fwd<T>, dim3((unsigned)lmin(tiles, 1 << 20)), dim3(LOOP_THREADS), 0, st, s, xt, w, b, yt, mean, rstd);
  }
  return rtg_launch_status();
}

template <class T>
int backward(const RtgLayerNormDesc* d, const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx,
             void* dw, void* db, float* ws, hipStream_t st) {
  const LnShape s = shape_of(d);
  const T *xt = reinterpret_cast<const T*>(x), *gt = reinterpret_cast<const T*>(dy);
  T* dt = reinterpret_cast<T*>(dx);
  const int slices = dw_slices(d);
  if (dx) {
    if (is_rows(d)) {
      RTG_KLAUNCH(ln_row_loop_dx<T>, dim3((unsigned)lmin(d->outer, 1 << 20)), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, w, dt);
    } else {
      const long long tiles = d->outer * ((d->inner + 63) / 64);
      RTG_KLAUNCH(ln_map_loop_dx<T>, dim3((unsigned)lmin(tiles, 1 << 20)), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, w, dt);
    }
    const int rc = rtg_launch_status();
    if (rc != RTG_OK) return rc;
  }
  if (!dw && !db) return RTG_OK;
  if (is_rows(d)) {
    RTG_KLAUNCH(ln_row_loop_dw<T>, dim3((unsigned)((d->n + 63) / 64), slices), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, ws, slices);
  } else {
    RTG_KLAUNCH(ln_map_loop_dw<T>, dim3((unsigned)lmin(d->n, 1 << 20), slices), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, ws, slices);
  }
  const int rc = rtg_launch_status();
  if (rc != RTG_OK) return rc;
  RTG_KLAUNCH(ln_finish, dim3((unsigned)rtg_ceil_div(d->n, FIN_COLS), 2), dim3(FIN_COLS * FIN_ROWS), 0, st, (const float*)ws, slices,
              d->n, dw, db, s.pbf);
  return rtg_launch_status();
}

}  // namespace

extern "C" int rtg_layernorm_forward(const RtgLayerNormDesc* d, const void* x, const void* weight, const void* bias, void* y,
                                     float* mean, float* rstd, void* stream) {
  const int rc = check_desc(d);
  if (rc != RTG_OK) return rc;
  if (d->outer == 0 || d->inner == 0) return RTG_OK;
  if (!x || !y || !mean != !rstd) return RTG_ENULL;
  return d->bf16 ? forward<rtg_bf16>(d, x, weight, bias, y, mean, rstd, (hipStream_t)stream)
                 : forward<float>(d, x, weight, bias, y, mean, rstd, (hipStream_t)stream);
}

extern "C" long long rtg_layernorm_ws(const RtgLayerNormDesc* d) {
  const int rc = check_desc(d);
  if (rc != RTG_OK) return rc;
  return 2 * d->n * dw_slices(d);
}

extern "C" int rtg_layernorm_backward(const RtgLayerNormDesc* d, const void* dy, const void* x, const float* mean, const float* rstd,
                                      const void* weight, void* dx, void* dweight, void* dbias, float* ws, void* stream) {
  const int rc = check_desc(d);
  if (rc != RTG_OK) return rc;
  const bool params = dweight || dbias;
  if (d->outer == 0 || d->inner == 0) {
    if (!params) return RTG_OK;
    RTG_KLAUNCH(ln_finish, dim3((unsigned)rtg_ceil_div(d->n, FIN_COLS), 2), dim3(FIN_COLS * FIN_ROWS), 0, (hipStream_t)stream,
                (const float*)nullptr, 0, d->n, dweight, dbias, d->param_bf16 != 0);
    return rtg_launch_status();
  }
  if (!dy || !x || !mean || !rstd || (params && !ws)) return RTG_ENULL;
  return d->bf16 ? backward<rtg_bf16>(d, dy, x, mean, rstd, weight, dx, dweight, dbias, ws, (hipStream_t)stream)
                 : backward<float>(d, dy, x, mean, rstd, weight, dx, dweight, dbias, ws, (hipStream_t)stream);
}

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
  float nf, inv_n, eps;                   // n, 1 / n
  int pbf;                                // weight / bias (and their gradients) are bf16
};

// sum / n: one multiplication and its correction by the remainder (what a division comes to, without its range checks: n is a
// plain number), so that the mean of equal values is that value
__device__ __forceinline__ float mean_of(float sum, const LnShape& s) {
  const float q = sum * s.inv_n, r = fmaf(-q, s.nf, sum);
  return isfinite(q) ? fmaf(r, s.inv_n, q) : q;
}
__device__ __forceinline__ float rstd_of(float sum, const LnShape& s) { return rsqrtf(sum * s.inv_n + s.eps); }

__device__ __forceinline__ float param_at(const void* p, int bf, long long i, float dflt) {
  if (!p) return dflt;
  return bf ? rtg_up(reinterpret_cast<const rtg_bf16*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}

// N parameters from index i on as floats (all of them exist); `dflt` where there are none
template <int N>
__device__ __forceinline__ void load_params(float (&out)[N], const void* p, int bf, long long i, float dflt) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = dflt;
  } else if (bf) {
    const rtg_bf16* q = reinterpret_cast<const rtg_bf16*>(p) + i;
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = rtg_up(q[e]);
  } else {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      RtgVec<float> v;
      v.load(reinterpret_cast<const float*>(p) + i + 4 * k);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * k + e] = v.get(e);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The register kernels.  All their accesses are whole vectors: where an axis ends inside a lane's vector, the lane's vector ends
// with the axis instead and repeats `dup` elements of the lane before it.  Those elements come out the same from both (each is
// computed from sums that everyone has in one order), so writing them twice is harmless; only sums leave the repeated ones out.
// A lane that lies behind the axis as a whole (dup >= N) loads what the last one loads and adds and writes nothing.
//
// Rows.  TPR threads hold a row in registers, VPT 16-byte vectors each, so x is read once; the sums are shuffles inside a wave
// and, for rows longer than a wave holds, one round through LDS each.  A block walks rows with the weights in registers and
// the next row's loads in flight while it works on this one.
// ---------------------------------------------------------------------------------------------------------------------
template <int K>
__device__ __forceinline__ void pin_all(float (&v)[K]) {
#pragma unroll
  for (int k = 0; k < K; ++k) rtg_pin(v[k]);
}

// sums of K values over the TPR threads of a row; `red`: K floats a wave, another buffer than the last call's (one barrier per
// call: a wave that writes this buffer again has passed the barrier of the call between)
template <int TPR, int BLK, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float (*red)[BLK / 64]) {
#pragma unroll
  for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], off, 64);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[k][wave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v[k] += red[k][first + i];
    }
  }
}

// the columns of a thread: vector k starts at col[k] and repeats dup[k] elements
template <int N, int TPR, int VPT>
struct RowLane {
  int col[VPT], dup[VPT];
  __device__ __forceinline__ RowLane(int t, int n) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int at = (k * TPR + t) * N;
      col[k] = at < n - N ? at : n - N;
      dup[k] = at - col[k];
    }
  }
};

// AHEAD 0 (rows of 1024 threads, 128 registers each): neither the weights nor the next row are held
template <class T, int TPR, int VPT, int BLK, int AHEAD>
__global__ __launch_bounds__(BLK) void ln_row_fwd(LnShape s, const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b,
                                                  T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  constexpr int N = RtgVec<T>::N, G = BLK / TPR;
  static_assert(TPR <= 64 || G == 1, "rows of several waves: one at a time, so that all threads meet at the barriers");
  __shared__ float red[2][1][BLK / 64];
  const int t = threadIdx.x % TPR;
  const RowLane<N, TPR, VPT> at(t, (int)s.n);
  const long long step = (long long)gridDim.x * G;
  long long row = (long long)blockIdx.x * G + threadIdx.x / TPR;
  if (row >= s.outer) return;                              // (whole groups; with barriers G is 1 and the grid no larger than the rows)
  RtgVec<T> v[VPT], next[VPT];
  float wr[AHEAD ? VPT : 1][N], br[AHEAD ? VPT : 1][N];
#pragma unroll
  for (int k = 0; k < VPT; ++k) next[k].load(x + row * s.xo + at.col[k]);
  if constexpr (AHEAD) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      load_params<N>(wr[k], w, s.pbf, at.col[k], 1.f);
      load_params<N>(br[k], b, s.pbf, at.col[k], 0.f);
    }
  }
  for (; row < s.outer; row += step) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) v[k] = next[k];
    const T* xn = x + (row + step < s.outer ? row + step : row) * s.xo;
    if constexpr (AHEAD) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) next[k].load(xn + at.col[k]);
    }
    float a[1] = {0.f};
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
#pragma unroll
      for (int e = 0; e < N; ++e) a[0] += e >= at.dup[k] ? v[k].get(e) : 0.f;
      rtg_pin(a[0]);
      v[k].hold();
    }
    row_sum<TPR, BLK, 1>(a, red[0]);
    const float mean = mean_of(a[0], s);
    a[0] = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = e >= at.dup[k] ? v[k].get(e) - mean : 0.f;
        a[0] += d * d;
      }
      rtg_pin(a[0]);
      v[k].hold();
    }
    row_sum<TPR, BLK, 1>(a, red[1]);
    const float rstd = rstd_of(a[0], s);
    T* yr = y + row * s.n;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      float o[N];
      if constexpr (!AHEAD) {
        load_params<N>(wr[0], w, s.pbf, at.col[k], 1.f);
        load_params<N>(br[0], b, s.pbf, at.col[k], 0.f);
      }
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = (v[k].get(e) - mean) * rstd * wr[AHEAD ? k : 0][e] + br[AHEAD ? k : 0][e];
      v[k].set(o);
      if (at.dup[k] < N) v[k].store(yr + at.col[k]);
    }
    if constexpr (!AHEAD) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) next[k].load(xn + at.col[k]);
    }
    if (mean_out && t == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

// dx, and the block's share of dw and db: a thread owns the same columns of every row its block walks, so their sums stay in
// registers; the groups of a block add theirs in LDS at the end, and ln_finish adds the blocks'.
template <class T, int TPR, int VPT, int BLK, int AHEAD>
__global__ __launch_bounds__(BLK) void ln_row_bwd(LnShape s, const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean_in,
                                                  const float* __restrict__ rstd_in, const void* __restrict__ w, T* __restrict__ dx,
                                                  float* __restrict__ part) {
  constexpr int N = RtgVec<T>::N, G = BLK / TPR, E = VPT * N;
  __shared__ float red[2][2][BLK / 64];
  __shared__ float sums[G > 1 ? E * BLK : 1];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const RowLane<N, TPR, VPT> at(t, (int)s.n);
  const long long step = (long long)gridDim.x * G, last = s.outer - 1;
  RtgVec<T> xv[VPT], gv[VPT], xn[AHEAD ? VPT : 1], gn[AHEAD ? VPT : 1];
  float mean, rstd, mean_n = 0.f, rstd_n = 0.f;
  const auto fetch = [&](RtgVec<T>* xd, RtgVec<T>* gd, float& m, float& r, long long row) __attribute__((always_inline)) {
    row = row < last ? row : last;                         // (a group behind the last row works on it once more, for nothing)
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      xd[k].load(x + row * s.xo + at.col[k]);
      gd[k].load(dy + row * s.n + at.col[k]);
    }
    m = mean_in[row];
    r = rstd_in[row];
  };
  long long base = (long long)blockIdx.x * G;
  if constexpr (AHEAD) fetch(xn, gn, mean_n, rstd_n, base + g);
  float wr[VPT][N], aw[VPT][N], ab[VPT][N];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    load_params<N>(wr[k], w, s.pbf, at.col[k], 1.f);
#pragma unroll
    for (int e = 0; e < N; ++e) aw[k][e] = ab[k][e] = 0.f;
  }
  int turn = 0;
  for (; base < s.outer; base += step, turn ^= 1) {
    const long long row = base + g;
    const int none = row <= last ? 0 : N;
    if constexpr (AHEAD) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        xv[k] = xn[k];
        gv[k] = gn[k];
      }
      mean = mean_n;
      rstd = rstd_n;
      fetch(xn, gn, mean_n, rstd_n, row + step);
    } else {
      fetch(xv, gv, mean, rstd, row);
    }
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int skip = at.dup[k] + none;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = e >= skip ? gv[k].get(e) : 0.f, h = e >= skip ? (xv[k].get(e) - mean) * rstd : 0.f, gw = d * wr[k][e];
        aw[k][e] += d * h;
        ab[k][e] += d;
        a[0] += gw;
        a[1] += gw * h;
      }
      pin_all<N>(aw[k]);
      pin_all<N>(ab[k]);
      pin_all<2>(a);
      gv[k].hold();
      xv[k].hold();
    }
    if (!dx) continue;
    row_sum<TPR, BLK, 2>(a, red[turn]);
    const float c1 = a[0] * s.inv_n, c2 = a[1] * s.inv_n;
    T* dr = dx + row * s.n;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = rstd * (gv[k].get(e) * wr[k][e] - c1 - (xv[k].get(e) - mean) * rstd * c2);
      xv[k].set(o);
      if (at.dup[k] + none < N) xv[k].store(dr + at.col[k]);
    }
  }
  if (!part) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = part + ((long long)blockIdx.x * 2 + which) * s.n;
    if constexpr (G == 1) {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (e >= at.dup[k]) out[at.col[k] + e] = which ? ab[k][e] : aw[k][e];
    } else {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) sums[(k * N + e) * BLK + threadIdx.x] = which ? ab[k][e] : aw[k][e];
      __syncthreads();
      for (int j = threadIdx.x; j < E * TPR; j += BLK) {
        const int k = j / (N * TPR), e = j / TPR % N, tt = j % TPR, nominal = (k * TPR + tt) * N, n = (int)s.n;
        const int col = nominal < n - N ? nominal : n - N;
        float a = 0.f;
        for (int i = 0; i < G; ++i) a += sums[(k * N + e) * BLK + i * TPR + tt];
        if (e >= nominal - col) out[col + e] = a;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Feature maps.  A wave holds a tile of LP * N adjacent positions (N in a lane's vector) with its 64 / LP channel lanes times
// CPT channels each in registers; W waves share the channels of a tile where one cannot hold them.  Every load is a whole
// 16 * LP bytes of a channel's row, CPT of them in flight per lane.
// ---------------------------------------------------------------------------------------------------------------------
// sums of K values per position over the channel lanes of a wave and the W waves of a team
template <int LP, int W, int K>
__device__ __forceinline__ void tile_sum(float (&v)[K], float (*red)[K * LP + 1]) {
#pragma unroll
  for (int off = LP; off < 64; off <<= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], off, 64);
  if constexpr (W > 1) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave / W * W;
    if (lane < LP)
#pragma unroll
      for (int k = 0; k < K; ++k) red[wave][k * LP + lane] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v[k] += red[first + i][k * LP + lane % LP];
    }
  }
}

constexpr int map_teams(int w) { return w < 4 ? 4 / w : 1; }
constexpr int map_block(int w) { return 64 * w * map_teams(w); }
template <class T, int LP, int W, int CPT>
struct MapTile {
  static constexpr int N = RtgVec<T>::N, CL = 64 / LP, TEAMS = map_teams(W), BLK = map_block(W);
  static constexpr int POS = LP * N, CH = CL * W * CPT;
};

template <int N>
__device__ __forceinline__ void store_floats(const float (&v)[N], float* p) {
#pragma unroll
  for (int k = 0; k < N / 4; ++k) {
    RtgVec<float> r;
    r.set({v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]});
    r.store(p + 4 * k);
  }
}

// where a lane of a tile stands.  The wave's part of every address is scalar, a lane's is 32 bits; a lane without a channel
// works on channel lane 0's (of the last channel, where the wave has none) for nothing
template <class T, int LP, int W, int CPT>
struct MapLane {
  using M = MapTile<T, LP, W, CPT>;
  int lane, wave, cw, n;                 // cw: the wave's first channel
  bool full;                             // every lane of the wave has CPT channels
  unsigned o, t;                         // clip, first position of the lane's vector
  int dup;
  __device__ __forceinline__ MapLane(const LnShape& s)
      : lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), cw(wave % W * M::CL), n((int)s.n),
        full(cw + (CPT - 1) * M::CL * W + M::CL <= n) {}
  __device__ __forceinline__ void go(const LnShape& s, unsigned tile, unsigned tiles, unsigned per) {
    const bool on = tile < tiles;        // (a team behind the last tile goes along to the barriers)
    o = on ? tile / per : 0;
    const int at = (int)((on ? tile - o * per : 0) * M::POS) + lane % LP * M::N, end = (int)s.inner - M::N;
    t = at < end ? at : end;
    dup = on ? at - (int)t : M::N;
  }
  __device__ __forceinline__ int channel(int i) const { return cw + i * M::CL * W + lane / LP; }
  __device__ __forceinline__ bool has(int i) const { return channel(i) < n; }
  __device__ __forceinline__ int base(int i) const { return cw + i * M::CL * W < n ? cw + i * M::CL * W : n - 1; }
  // byte offset of the lane behind its wave's channel; of channel lane 0
  __device__ __forceinline__ unsigned off(long long stride) const {
    return (t + (unsigned)(lane / LP) * (unsigned)stride) * (unsigned)sizeof(T);
  }
  __device__ __forceinline__ unsigned off0() const { return t * (unsigned)sizeof(T); }
  __device__ __forceinline__ static T* byte(T* p, unsigned off) { return reinterpret_cast<T*>(reinterpret_cast<char*>(p) + off); }
  __device__ __forceinline__ static const T* byte(const T* p, unsigned off) {
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + off);
  }
  __device__ __forceinline__ void load(RtgVec<T> (&v)[CPT], const T* p, long long outer, long long stride) const {
    p += o * outer;
    if (full) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) v[i].load(byte(p + (cw + i * M::CL * W) * stride, off(stride)));
    } else {
#pragma unroll
      for (int i = 0; i < CPT; ++i) v[i].load(byte(p + base(i) * stride, has(i) ? off(stride) : off0()));
#pragma unroll
      for (int i = 0; i < CPT; ++i)
        if (!has(i)) v[i].zero();
    }
  }
  // f(i) -> vector i, for the lanes that own it
  template <class F>
  __device__ __forceinline__ void store(T* p, long long outer, long long stride, F f) const {
    p += o * outer;
    if (dup >= M::N) return;
    if (full) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) f(i).store(byte(p + (cw + i * M::CL * W) * stride, off(stride)));
    } else {
#pragma unroll
      for (int i = 0; i < CPT; ++i)
        if (has(i)) f(i).store(byte(p + base(i) * stride, off(stride)));
    }
  }
  __device__ __forceinline__ void params(float (&out)[CPT], const void* p, int bf, float dflt) const {
    if (!p) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) out[i] = dflt;
    } else if (bf) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) out[i] = rtg_up(reinterpret_cast<const rtg_bf16*>(p)[has(i) ? channel(i) : 0]);
    } else {
#pragma unroll
      for (int i = 0; i < CPT; ++i) out[i] = reinterpret_cast<const float*>(p)[has(i) ? channel(i) : 0];
    }
  }
};

template <class T, int LP, int W, int CPT>
__global__ __launch_bounds__(map_block(W)) void ln_map_fwd(LnShape s, const T* __restrict__ x, const void* __restrict__ w,
                                                                           const void* __restrict__ b, T* __restrict__ y,
                                                                           float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  using M = MapTile<T, LP, W, CPT>;
  constexpr int N = M::N;
  __shared__ float red[2][W > 1 ? M::BLK / 64 : 1][N * LP + 1];
  MapLane<T, LP, W, CPT> at(s);
  const unsigned per = (unsigned)((s.inner + M::POS - 1) / M::POS);
  at.go(s, blockIdx.x * M::TEAMS + at.wave / W, (unsigned)s.outer * per, per);
  RtgVec<T> v[CPT];
  at.load(v, x, s.xo, s.xn);
  float wr[CPT], br[CPT], a[N], mean[N], rstd[N];
  at.params(wr, w, s.pbf, 1.f);
  at.params(br, b, s.pbf, 0.f);
#pragma unroll
  for (int e = 0; e < N; ++e) a[e] = 0.f;
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] += v[i].get(e);
    pin_all<N>(a);
    v[i].hold();
  }
  tile_sum<LP, W, N>(a, red[0]);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    mean[e] = mean_of(a[e], s);
    a[e] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = at.has(i) ? v[i].get(e) - mean[e] : 0.f;
      a[e] += d * d;
    }
    pin_all<N>(a);
    v[i].hold();
  }
  tile_sum<LP, W, N>(a, red[1]);
#pragma unroll
  for (int e = 0; e < N; ++e) rstd[e] = rstd_of(a[e], s);
  at.store(y, s.n * s.inner, s.inner, [&](int i) __attribute__((always_inline)) {
    float r[N];
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = (v[i].get(e) - mean[e]) * rstd[e] * wr[i] + br[i];
    v[i].set(r);
    return v[i];
  });
  if (mean_out && at.wave % W == 0 && at.lane < LP && at.dup < N) {
    store_floats<N>(mean, mean_out + at.o * s.inner + at.t);
    store_floats<N>(rstd, rstd_out + at.o * s.inner + at.t);
  }
}

// dx and the team's share of dw, db: a lane adds its channels' products over its positions and over the tiles its team walks;
// the position lanes meet in shuffles at the end, the teams of a block in LDS
template <class T, int LP, int W, int CPT>
__global__ __launch_bounds__(map_block(W)) void ln_map_bwd(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                                           const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                           const void* __restrict__ w, T* __restrict__ dx,
                                                                           float* __restrict__ part) {
  using M = MapTile<T, LP, W, CPT>;
  constexpr int N = M::N;
  __shared__ float red[2][W > 1 ? M::BLK / 64 : 1][2 * N * LP + 1];
  __shared__ float sums[2][M::TEAMS][M::CH];
  MapLane<T, LP, W, CPT> at(s);
  const int team = at.wave / W;
  const unsigned per = (unsigned)((s.inner + M::POS - 1) / M::POS), tiles = (unsigned)s.outer * per;
  float wr[CPT], aw[CPT], ab[CPT];
  at.params(wr, w, s.pbf, 1.f);
#pragma unroll
  for (int i = 0; i < CPT; ++i) aw[i] = ab[i] = 0.f;
  int turn = 0;
  for (unsigned base = blockIdx.x * M::TEAMS; base < tiles; base += gridDim.x * M::TEAMS, turn ^= 1) {
    at.go(s, base + team, tiles, per);
    RtgVec<T> xv[CPT], gv[CPT];
    at.load(xv, x, s.xo, s.xn);
    at.load(gv, dy, s.n * s.inner, s.inner);
    float mean[N], rstd[N], a[2 * N];
    load_params<N>(mean, mean_in, 0, at.o * s.inner + at.t, 0.f);
    load_params<N>(rstd, rstd_in, 0, at.o * s.inner + at.t, 0.f);
#pragma unroll
    for (int e = 0; e < 2 * N; ++e) a[e] = 0.f;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = gv[i].get(e), h = (xv[i].get(e) - mean[e]) * rstd[e], gw = d * wr[i], once = e >= at.dup ? d : 0.f;
        aw[i] += once * h;
        ab[i] += once;
        a[e] += gw;
        a[N + e] += gw * h;
      }
      rtg_pin(aw[i]);
      rtg_pin(ab[i]);
      pin_all<2 * N>(a);
      gv[i].hold();
      xv[i].hold();
    }
    if (!dx) continue;
    tile_sum<LP, W, 2 * N>(a, red[turn]);
#pragma unroll
    for (int e = 0; e < 2 * N; ++e) a[e] *= s.inv_n;
    at.store(dx, s.n * s.inner, s.inner, [&](int i) __attribute__((always_inline)) {
      float r[N];
#pragma unroll
      for (int e = 0; e < N; ++e)
        r[e] = rstd[e] * (gv[i].get(e) * wr[i] - a[e] - (xv[i].get(e) - mean[e]) * rstd[e] * a[N + e]);
      xv[i].set(r);
      return xv[i];
    });
  }
  if (!part) return;
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
#pragma unroll
    for (int off = 1; off < LP; off <<= 1) {
      aw[i] += __shfl_xor(aw[i], off, 64);
      ab[i] += __shfl_xor(ab[i], off, 64);
    }
    if (at.lane % LP == 0) {
      sums[0][team][at.channel(i)] = aw[i];
      sums[1][team][at.channel(i)] = ab[i];
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * M::CH; j += M::BLK) {
    const int which = j / M::CH, c = j % M::CH;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < M::TEAMS; ++i) v += sums[which][i][c];
    if (c < at.n) part[((long long)blockIdx.x * 2 + which) * s.n + c] = v;
  }
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
    const float mean = mean_of(rtg_block_sum(acc, red), s);
    acc = 0.f;
    for (long long i = threadIdx.x; i < s.n; i += LOOP_THREADS) {
      const float d = rtg_up(xr[i]) - mean;
      acc += d * d;
    }
    const float rstd = rstd_of(rtg_block_sum(acc, red), s);
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
    const float c1 = rtg_block_sum(a1, red) * s.inv_n, c2 = rtg_block_sum(a2, red) * s.inv_n;
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
    const float mean = mean_of(wave_column_sum(acc, red), s);
    acc = 0.f;
    if (in)
      for (long long c = wave; c < s.n; c += 4) {
        const float d = rtg_up(xp[c * s.xn]) - mean;
        acc += d * d;
      }
    const float rstd = rstd_of(wave_column_sum(acc, red), s);
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
    const float c1 = wave_column_sum(a1, red) * s.inv_n, c2 = wave_column_sum(a2, red) * s.inv_n;
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
  return LnShape{d->outer, d->n, d->inner, d->x_outer, d->x_n, (float)d->n, (float)(1.0 / (double)d->n), d->eps, d->param_bf16 != 0};
}

bool is_rows(const RtgLayerNormDesc* d) { return d->inner == 1; }

// What serves a problem: the smallest register tile that holds the normalised axis, else the kernels for any size.  `tile` is
// the tile's number in the dispatch below, `blocks` the grid, in the backward also the number of partial dw / db.
struct Plan { int tile; int blocks; };
constexpr int LOOPS = -1;

// rows: threads per row and 16-byte vectors per thread.  Rows of up to 64 vectors leave no lane of a group idle for the sake of
// a shuffle tree; past four vectors a thread (the weights' registers) a row goes to a whole block.
struct RowTile { int tpr, vpt; };
constexpr RowTile FWD_TILES[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {1024, 2}, {1024, 4}};
// backward: sixteen elements a thread (weight, dw and db are three registers each)
constexpr RowTile BWD_F32[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {512, 4}, {1024, 3}};
constexpr RowTile BWD_BF16[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {256, 1}, {256, 2}, {512, 2}, {1024, 2}, {1024, 2}};

int row_tile(const RowTile* tiles, long long n, int bf16) {
  const int vec = bf16 ? 8 : 4;
  if (n < vec) return LOOPS;
  const long long nv = (n + vec - 1) / vec;
  for (int i = 0; i < 10; ++i)
    if (nv <= tiles[i].tpr * tiles[i].vpt) return i;
  return LOOPS;
}

// maps: position lanes, waves that share the channels, channels a lane (backward: x and dy are both held, eight channels a lane)
struct MapCfg { int lp, w, cpt; };
constexpr MapCfg MAP_FWD[] = {{2, 1, 4}, {2, 1, 16}, {2, 2, 16}, {32, 1, 8}, {8, 1, 4}, {8, 1, 8}, {8, 1, 16}, {8, 2, 16}, {8, 4, 16}, {8, 8, 16}};
constexpr MapCfg MAP_BWD[] = {{2, 1, 4}, {2, 1, 8}, {2, 2, 8}, {2, 4, 8}, {32, 1, 8}, {8, 1, 4}, {8, 1, 8}, {8, 2, 8}, {8, 4, 8}, {8, 8, 8}, {4, 8, 8}};

struct MapPlan { int i; long long blocks; };               // blocks: enough for one tile a team
template <int COUNT>
MapPlan map_tile(const MapCfg (&cfg)[COUNT], const RtgLayerNormDesc* d) {
  const int vec = d->bf16 ? 8 : 4;
  if (d->inner < vec || d->inner >= 1 << 24 || d->x_n >= 1 << 24) return {LOOPS, 0};      // (a lane's offset in a tile has 32 bits)
  for (int i = 0; i < COUNT; ++i) {
    const MapCfg& m = cfg[i];
    if (m.lp == 2 ? d->inner > 2 * vec : d->inner <= 2 * vec) continue;
    if (m.lp == 32 && d->inner < 32 * vec) continue;       // few channels and many positions: more positions a wave
    if (d->n > 64 / m.lp * m.w * m.cpt) continue;
    const long long pos = m.lp * vec, tiles = d->outer * ((d->inner + pos - 1) / pos), teams = map_teams(m.w);
    if (tiles >= 1ll << 30) return {LOOPS, 0};
    return {i, (tiles + teams - 1) / teams};
  }
  return {LOOPS, 0};
}

// blocks for `items` tiles of work, at most `cap` of them with as even a share as can be
int even_blocks(long long items, long long cap) {
  const long long rounds = (items + cap - 1) / cap;
  return (int)((items + rounds - 1) / rounds);
}

constexpr int row_block(int tpr) { return tpr <= 256 ? 256 : tpr; }
constexpr int row_block_bwd(int tpr) { return tpr <= 512 ? 512 : tpr; }

Plan plan_fwd(const RtgLayerNormDesc* d) {
  if (is_rows(d)) {
    const int i = row_tile(FWD_TILES, d->n, d->bf16);
    if (i == LOOPS) return {LOOPS, (int)lmin(d->outer, 1 << 20)};
    const int blk = row_block(FWD_TILES[i].tpr), groups = blk / FWD_TILES[i].tpr;
    return {i, even_blocks((d->outer + groups - 1) / groups, 256 * (2048 / blk))};
  }
  const MapPlan m = map_tile(MAP_FWD, d);
  if (m.i == LOOPS) return {LOOPS, (int)lmin(d->outer * ((d->inner + 63) / 64), 1 << 20)};
  return {m.i, (int)m.blocks};
}

Plan plan_bwd(const RtgLayerNormDesc* d) {
  if (is_rows(d)) {
    const RowTile* tiles = d->bf16 ? BWD_BF16 : BWD_F32;
    const int i = row_tile(tiles, d->n, d->bf16);
    if (i != LOOPS) {
      const int blk = row_block_bwd(tiles[i].tpr), groups = blk / tiles[i].tpr;
      return {i, even_blocks((d->outer + groups - 1) / groups, 512)};
    }
    const long long cols = (d->n + 63) / 64, s = lmin((d->outer + 15) / 16, (2048 + cols - 1) / cols);
    return {LOOPS, (int)(s < 1 ? 1 : lmin(s, 1024))};
  }
  const MapPlan m = map_tile(MAP_BWD, d);
  if (m.i != LOOPS) return {m.i, even_blocks(m.blocks, MAP_BWD[m.i].w > 4 ? 256 : 512)};
  const long long s = lmin((d->outer * d->inner + 1023) / 1024, (2048 + d->n - 1) / d->n);
  return {LOOPS, (int)(s < 1 ? 1 : lmin(s, 1024))};
}

template <class T>
int forward(const RtgLayerNormDesc* d, const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, hipStream_t st) {
  const LnShape s = shape_of(d);
  const T* xt = reinterpret_cast<const T*>(x);
  T* yt = reinterpret_cast<T*>(y);
  const Plan p = plan_fwd(d);
#define LN_ROW(I, TPR, VPT)                                                                                                  \
  case I:                                                                                                                    \
    RTG_KLAUNCH((ln_row_fwd<T, TPR, VPT, row_block(TPR), (TPR * VPT < 4096)>), dim3(p.blocks), dim3(row_block(TPR)), 0, st, s, xt, \
                w, b, yt, mean, rstd);                                                                                       \
    return rtg_launch_status()
#define LN_MAP(I, LP, W, CPT)                                                                                                \
  case I:                                                                                                                    \
    RTG_KLAUNCH((ln_map_fwd<T, LP, W, CPT>), dim3(p.blocks), dim3(map_block(W)), 0, st, s, xt, w, b, yt, mean, rstd); \
    return rtg_launch_status()
  if (is_rows(d)) {
    switch (p.tile) {
      LN_ROW(0, 8, 1);
      LN_ROW(1, 16, 1);
      LN_ROW(2, 32, 1);
      LN_ROW(3, 64, 1);
      LN_ROW(4, 64, 2);
      LN_ROW(5, 64, 4);
      LN_ROW(6, 256, 2);
      LN_ROW(7, 256, 4);
      LN_ROW(8, 1024, 2);
      LN_ROW(9, 1024, 4);
    }
    RTG_KLAUNCH(ln_row_loop_fwd<T>, dim3(p.blocks), dim3(LOOP_THREADS), 0, st, s, xt, w, b, yt, mean, rstd);
  } else {
    switch (p.tile) {
      LN_MAP(0, 2, 1, 4);
      LN_MAP(1, 2, 1, 16);
      LN_MAP(2, 2, 2, 16);
      LN_MAP(3, 32, 1, 8);
      LN_MAP(4, 8, 1, 4);
      LN_MAP(5, 8, 1, 8);
      LN_MAP(6, 8, 1, 16);
      LN_MAP(7, 8, 2, 16);
      LN_MAP(8, 8, 4, 16);
      LN_MAP(9, 8, 8, 16);
    }
    RTG_KLAUNCH(ln_map_loop_fwd<T>, dim3(p.blocks), dim3(LOOP_THREADS), 0, st, s, xt, w, b, yt, mean, rstd);
  }
#undef LN_ROW
#undef LN_MAP
  return rtg_launch_status();
}

template <class T>
int backward(const RtgLayerNormDesc* d, const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx,
             void* dw, void* db, float* ws, hipStream_t st) {
  const LnShape s = shape_of(d);
  const T *xt = reinterpret_cast<const T*>(x), *gt = reinterpret_cast<const T*>(dy);
  T* dt = reinterpret_cast<T*>(dx);
  const bool params = dw || db;
  if (!dx && !params) return RTG_OK;
  float* const part = params ? ws : nullptr;
  const Plan p = plan_bwd(d);
#define LN_ROW(I, TPR, VPT, AHEAD)                                                                                           \
  case I:                                                                                                                    \
    RTG_KLAUNCH((ln_row_bwd<T, TPR, VPT, row_block_bwd(TPR), AHEAD>), dim3(p.blocks), dim3(row_block_bwd(TPR)), 0, st, s, gt, \
                xt, mean, rstd, w, dt, part);                                                                                \
    break
#define LN_MAP(I, LP, W, CPT)                                                                                                \
  case I:                                                                                                                    \
    RTG_KLAUNCH((ln_map_bwd<T, LP, W, CPT>), dim3(p.blocks), dim3(map_block(W)), 0, st, s, gt, xt, mean, rstd, w, dt, part); \
    break
  constexpr bool BF = sizeof(T) == 2;
  if (is_rows(d) && p.tile != LOOPS) {
    switch (p.tile) {
      LN_ROW(0, 8, 1, 1);
      LN_ROW(1, 16, 1, 1);
      LN_ROW(2, 32, 1, 1);
      LN_ROW(3, 64, 1, 1);
      LN_ROW(4, 64, 2, 1);
      LN_ROW(5, (BF ? 256 : 64), (BF ? 1 : 4), 1);
      LN_ROW(6, 256, 2, 1);
      LN_ROW(7, (BF ? 512 : 256), (BF ? 2 : 4), 1);
      LN_ROW(8, (BF ? 1024 : 512), (BF ? 2 : 4), (BF ? 0 : 1));
      LN_ROW(9, 1024, (BF ? 2 : 3), 0);
    }
  } else if (is_rows(d)) {
    if (dx) {
      RTG_KLAUNCH(ln_row_loop_dx<T>, dim3((unsigned)lmin(d->outer, 1 << 20)), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, w, dt);
      const int rc = rtg_launch_status();
      if (rc != RTG_OK) return rc;
    }
    if (params)
      RTG_KLAUNCH(ln_row_loop_dw<T>, dim3((unsigned)((d->n + 63) / 64), p.blocks), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, part, p.blocks);
  } else if (p.tile != LOOPS) {
    switch (p.tile) {
      LN_MAP(0, 2, 1, 4);
      LN_MAP(1, 2, 1, 8);
      LN_MAP(2, 2, 2, 8);
      LN_MAP(3, 2, 4, 8);
      LN_MAP(4, 32, 1, 8);
      LN_MAP(5, 8, 1, 4);
      LN_MAP(6, 8, 1, 8);
      LN_MAP(7, 8, 2, 8);
      LN_MAP(8, 8, 4, 8);
      LN_MAP(9, 8, 8, 8);
      LN_MAP(10, 4, 8, 8);
    }
  } else {
    if (dx) {
      const long long tiles = d->outer * ((d->inner + 63) / 64);
      RTG_KLAUNCH(ln_map_loop_dx<T>, dim3((unsigned)lmin(tiles, 1 << 20)), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, w, dt);
      const int rc = rtg_launch_status();
      if (rc != RTG_OK) return rc;
    }
    if (params)
      RTG_KLAUNCH(ln_map_loop_dw<T>, dim3((unsigned)lmin(d->n, 1 << 20), p.blocks), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, part, p.blocks);
  }
#undef LN_ROW
#undef LN_MAP
  const int rc = rtg_launch_status();
  if (rc != RTG_OK || !params) return rc;
  RTG_KLAUNCH(ln_finish, dim3((unsigned)rtg_ceil_div(d->n, FIN_COLS), 2), dim3(FIN_COLS * FIN_ROWS), 0, st, (const float*)ws, p.blocks,
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
  return d->outer && d->inner ? 2 * d->n * plan_bwd(d).blocks : 1;
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

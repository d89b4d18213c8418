// rtg_layernorm.hip — layer norm forward and backward over the last axis (rows) or over the channel axis of feature maps
// (see include/rtg.h, rtg_layernorm_*).
//
//   y = (x - mean) * rstd * w + b                                    per row: mean, var over n elements
//   g = dy * w;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat));  dw = sum dy * xhat;  db = sum dy
//
// ~8 (forward) and ~16 (backward) operations per element of 4 .. 12 bytes moved: bound by HBM, which the large problems reach:
// 16384 x 4096 bf16 45.8 us forward (5.9 TB/s) and 75 backward (5.4), floats 83 (6.5) and 129 (6.2); a map of (32, 128, 16384)
// floats 83 and 144; a token's row of 4096 3.4 us and a launch of nothing 2.8.
#include "rtg_vec.h"

namespace {

constexpr int LOOP_THREADS = 1024;
constexpr int FIN_COLS = 32, FIN_ROWS = 32;

struct LnShape {
  long long outer, n, inner, xo, xn;      // x[o * xo + c * xn + t]; everything else contiguous
  float nf, inv_n, eps;                   // n, 1 / n
  int pbf;                                // weight / bias (and their gradients) are bf16
  int once;                               // what is read goes by the caches: below
};

// What a kernel reads goes by the caches where that much is not in the memory-side cache (256 MB) when somebody reads it next:
// 16384 x 4096 floats 95 -> 83 us forward, 154 -> 129 backward, (32, 128, 16384) floats 109 -> 83 and 171 -> 144; of 64 MB it
// costs up to a tenth, a neighbour's part of a shared line comes twice then.
constexpr long long CACHED = 256ll << 20;
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

__device__ __forceinline__ void put_param(void* p, int bf, long long i, float v) {
  if (!p) return;
  if (bf) rtg_down(v, reinterpret_cast<rtg_bf16*>(p)[i]);
  else reinterpret_cast<float*>(p)[i] = v;
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
  } else if constexpr (N == 1) {
    out[0] = reinterpret_cast<const float*>(p)[i];
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

template <int N>
__device__ __forceinline__ void store_floats(const float (&v)[N], float* p) {
  if constexpr (N == 1) *p = v[0];
#pragma unroll
  for (int k = 0; k < N / 4; ++k) {
    RtgVec<float> r;
    r.set({v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]});
    r.store(p + 4 * k);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The register kernels.  All their accesses are whole vectors: where an axis ends inside a lane's vector, the lane's vector ends
// with the axis instead and repeats `dup` elements of the lane before it.  Those elements come out the same from both (each is
// computed from sums that everyone has in one order), so writing them twice is harmless; only sums leave the repeated ones out.
// A lane that lies behind the axis as a whole (dup >= N) loads what the last one loads and adds and writes nothing.
//
// Rows.  TPR threads hold a row in registers, VPT 16-byte vectors each, so x is read once; the sums are lane swaps inside a wave
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
  for (int k = 0; k < K; ++k) v[k] = rtg_group_sum<(TPR < 64 ? TPR : 64)>(v[k]);
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
template <class T, int TPR, int VPT, int BLK, int AHEAD, bool ONCE>
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
  for (int k = 0; k < VPT; ++k) rtg_load<ONCE>(next[k], x + row * s.xo + at.col[k]);
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
      for (int k = 0; k < VPT; ++k) rtg_load<ONCE>(next[k], xn + at.col[k]);
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
      for (int k = 0; k < VPT; ++k) rtg_load<ONCE>(next[k], xn + at.col[k]);
    }
    if (mean_out && t == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

// dx, and the block's share of dw and db: a thread owns the same columns of every row its block walks, so their sums stay in
// registers; the groups of a block add theirs in LDS at the end, and ln_finish adds the blocks'.
template <class T, int TPR, int VPT, int BLK, int AHEAD, bool ONCE>
__global__ __launch_bounds__(BLK) void ln_row_bwd(LnShape s, const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean_in,
                                                  const float* __restrict__ rstd_in, const void* __restrict__ w, T* __restrict__ dx,
                                                  float* __restrict__ part, void* __restrict__ dw, void* __restrict__ db) {
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
      rtg_load<ONCE>(xd[k], x + row * s.xo + at.col[k]);
      rtg_load<ONCE>(gd[k], dy + row * s.n + at.col[k]);
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
    float* const out = part + ((long long)blockIdx.x * 2 + which) * s.n;
    if constexpr (G > 1) {
      // (the column order of the vectors, so that both sides of the exchange go through LDS in adjacent words)
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) sums[g * (TPR * E) + (k * TPR + t) * N + e] = which ? ab[k][e] : aw[k][e];
      __syncthreads();
      for (int j = threadIdx.x; j < TPR * E; j += BLK) {
        const int at0 = j / N * N, n = (int)s.n, col = at0 < n - N ? at0 : n - N;
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i) a += sums[i * (TPR * E) + j];
        if (j % N < at0 - col) continue;
        if (gridDim.x > 1) out[col + j % N] = a;
        else put_param(which ? db : dw, s.pbf, col + j % N, a);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        float(&v)[N] = which ? ab[k] : aw[k];
        if (gridDim.x > 1 && at.dup[k] == 0) {
          store_floats<N>(v, out + at.col[k]);
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (e >= at.dup[k]) {
              if (gridDim.x > 1) out[at.col[k] + e] = v[e];
              else put_param(which ? db : dw, s.pbf, at.col[k] + e, v[e]);
            }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Feature maps.  A wave holds a tile of LP * N adjacent positions (N in a lane's vector) with its 64 / LP channel lanes times
// CPT channels each in registers; W waves share the channels of a tile where one cannot hold them.  Every load is a whole
// 16 * LP bytes of a channel's row, CPT of them in flight per lane: (32, 128, 2048) floats 12.0 us forward (5.6 TB/s), 24 backward;
// (16, 512, 1025), whose channels start anywhere in a line, 13.7 and 28.8 with the join of dw and db.
// ---------------------------------------------------------------------------------------------------------------------
// workgroup b of a grid of 8 k runs on XCD b % 8 (each has its own L2): neighbours in the order of the tiles are put on one XCD, so
// a line that two tiles share — rows of a map that do not start on a line — is fetched once
__device__ __forceinline__ unsigned xcd_order(unsigned b, unsigned grid) { return b % 8 * (grid / 8) + b / 8; }

// K sums over the channel lanes of a wave and the W waves of a team, scattered over the lanes (rtg_scatter_sum)
template <int LP, int W, int K>
__device__ __forceinline__ void tile_sum(float (&v)[K], float (*red)[64 * rtg_scattered(LP, K)]) {
  constexpr int R = rtg_scattered(LP, K);
  rtg_scatter_sum<LP, K>(v);
  if constexpr (W > 1) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave / W * W;
#pragma unroll
    for (int k = 0; k < R; ++k) red[wave][k * 64 + lane] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < R; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v[k] += red[first + i][k * 64 + lane];
    }
  }
}

constexpr int map_teams(int w) { return w < 4 ? 4 / w : 1; }
constexpr int map_block(int w) { return 64 * w * map_teams(w); }
template <class V, int LP, int W, int CPT>
struct MapTile {
  static constexpr int N = V::N, CL = 64 / LP, TEAMS = map_teams(W), BLK = map_block(W);
  static constexpr int POS = LP * N, CH = CL * W * CPT;
};

// where a lane of a tile stands.  The wave's part of every address is scalar, a lane's is 32 bits; a lane without a channel
// works on channel lane 0's (of the last channel, where the wave has none) for nothing
template <class V, int LP, int W, int CPT>
struct MapLane {
  using T = typename V::T;
  using M = MapTile<V, LP, W, CPT>;
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
  // f(i) -> where vector i lies.  The fences keep the branches apart (merged, the loads would be of the plain kind); a loop that
  // has the next loads in flight cannot take such a branch, so the row kernels are built both ways
  __device__ __forceinline__ static void fence() { asm volatile("" ::: "memory"); }
  template <class F>
  __device__ __forceinline__ static void fetch(V (&v)[CPT], int once, F f) {
    if (once) {
      fence();
#pragma unroll
      for (int i = 0; i < CPT; ++i) v[i].load_once(f(i));
      fence();
    } else {
#pragma unroll
      for (int i = 0; i < CPT; ++i) v[i].load(f(i));
    }
  }
  __device__ __forceinline__ void load(V (&v)[CPT], const T* p, long long outer, long long stride, int once) const {
    p += o * outer;
    if (full) {
      fetch(v, once, [&](int i) __attribute__((always_inline)) { return byte(p + (cw + i * M::CL * W) * stride, off(stride)); });
    } else {
      fetch(v, once, [&](int i) __attribute__((always_inline)) { return byte(p + base(i) * stride, has(i) ? off(stride) : off0()); });
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

template <class V, int LP, int W, int CPT, class T = typename V::T>
__global__ __launch_bounds__(map_block(W)) void ln_map_fwd(LnShape s, const T* __restrict__ x, const void* __restrict__ w,
                                                                           const void* __restrict__ b, T* __restrict__ y,
                                                                           float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                                           unsigned first) {
  using M = MapTile<V, LP, W, CPT>;
  constexpr int N = M::N;
  constexpr int R = rtg_scattered(LP, N);
  __shared__ float red[2][W > 1 ? M::BLK / 64 : 1][64 * R];
  MapLane<V, LP, W, CPT> at(s);
  const unsigned per = (unsigned)((s.inner + M::POS - 1) / M::POS);
  at.go(s, (first + xcd_order(blockIdx.x, gridDim.x)) * M::TEAMS + at.wave / W, (unsigned)s.outer * per, per);
  V v[CPT];
  at.load(v, x, s.xo, s.xn, s.once);
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
  for (int k = 0; k < R; ++k) mean[k] = mean_of(a[k], s);
  rtg_gather<LP, N>(mean);
#pragma unroll
  for (int e = 0; e < N; ++e) a[e] = 0.f;
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
  for (int k = 0; k < R; ++k) rstd[k] = rstd_of(a[k], s);
  rtg_gather<LP, N>(rstd);
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
template <class V, int LP, int W, int CPT, class T = typename V::T>
__global__ __launch_bounds__(map_block(W)) void ln_map_bwd(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                                           const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                                           const void* __restrict__ w, T* __restrict__ dx,
                                                                           float* __restrict__ part) {
  using M = MapTile<V, LP, W, CPT>;
  constexpr int N = M::N;
  constexpr int R = rtg_scattered(LP, 2 * N);
  __shared__ float red[2][W > 1 ? M::BLK / 64 : 1][64 * R];
  __shared__ float sums[2][M::TEAMS][M::CH];
  MapLane<V, LP, W, CPT> at(s);
  const int team = at.wave / W;
  const unsigned per = (unsigned)((s.inner + M::POS - 1) / M::POS), tiles = (unsigned)s.outer * per;
  float wr[CPT], aw[CPT], ab[CPT];
  at.params(wr, w, s.pbf, 1.f);
#pragma unroll
  for (int i = 0; i < CPT; ++i) aw[i] = ab[i] = 0.f;
  int turn = 0;
  for (unsigned base = xcd_order(blockIdx.x, gridDim.x) * M::TEAMS; base < tiles; base += gridDim.x * M::TEAMS, turn ^= 1) {
    at.go(s, base + team, tiles, per);
    V xv[CPT], gv[CPT];
    at.load(xv, x, s.xo, s.xn, s.once);
    at.load(gv, dy, s.n * s.inner, s.inner, s.once);
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
    for (int k = 0; k < R; ++k) a[k] *= s.inv_n;
    rtg_gather<LP, 2 * N>(a);
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
// Kernels for any size.  A row or a column of channels that no register kernel holds is read once per sum (the later reads
// come from L2 or the memory-side cache): 1000 rows of 40000 floats 97 us forward, 194 backward (3.3 and 2.5 TB/s of what has to
// move).  ln_tiny serves rows of less than a vector, a thread each (1000000 x 3 floats 8.9 and 14.1 us, 1000000 x 7 bf16 values
// 14.9 and 24.6, and 4 for the join: 2.4 .. 3.6 and 2.0 .. 3.1 TB/s of what has to move).
// ---------------------------------------------------------------------------------------------------------------------
template <int BLK>
__device__ __forceinline__ float loop_sum(float v, float* red) {
  v = rtg_group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < BLK / 64; ++i) v += red[i];
  return v;
}

// f(first element, vector of x, vector of g) for the whole vectors of a row, f(element, x, g) for those behind them; x or g alone
// where the other is the same pointer
template <class T, class F>
__device__ __forceinline__ void row_walk(const T* x, const T* g, long long n, F f) {
  constexpr int N = RtgVec<T>::N;
  const long long nv = n / N;
#pragma unroll 2
  for (long long i = threadIdx.x; i < nv; i += LOOP_THREADS) {
    RtgVec<T> a, b;
    a.load(x + i * N);
    b.load(g + i * N);
    float xv[N], gv[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      xv[e] = a.get(e);
      gv[e] = b.get(e);
    }
    f(i * N, xv, gv);
  }
  if (nv * N + threadIdx.x < n) {
    const float xv[1] = {rtg_up(x[nv * N + threadIdx.x])}, gv[1] = {rtg_up(g[nv * N + threadIdx.x])};
    f(nv * N + threadIdx.x, xv, gv);
  }
}
template <class T, int K>
__device__ __forceinline__ void put_row(const float (&v)[K], T* p) {
  if constexpr (K == 1) {
    rtg_down(v[0], *p);
  } else {
    RtgVec<T> r;
    r.set(v);
    r.store(p);
  }
}

template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_row_loop_fwd(LnShape s, const T* __restrict__ x, const void* __restrict__ w,
                                                                const void* __restrict__ b, T* __restrict__ y,
                                                                float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float red[LOOP_THREADS / 64];
  for (long long row = blockIdx.x; row < s.outer; row += gridDim.x) {
    const T* xr = x + row * s.xo;
    T* yr = y + row * s.n;
    float acc = 0.f;
    row_walk(xr, xr, s.n, [&](long long, auto& v, auto&) __attribute__((always_inline)) {
#pragma unroll
      for (float e : v) acc += e;
    });
    const float mean = mean_of(loop_sum<LOOP_THREADS>(acc, red), s);
    acc = 0.f;
    row_walk(xr, xr, s.n, [&](long long, auto& v, auto&) __attribute__((always_inline)) {
#pragma unroll
      for (float e : v) acc += (e - mean) * (e - mean);
    });
    const float rstd = rstd_of(loop_sum<LOOP_THREADS>(acc, red), s);
    row_walk(xr, xr, s.n, [&](long long i, auto& v, auto&) __attribute__((always_inline)) {
      constexpr int K = sizeof(v) / sizeof(float);
      float wr[K], br[K], o[K];
      load_params<K>(wr, w, s.pbf, i, 1.f);
      load_params<K>(br, b, s.pbf, i, 0.f);
#pragma unroll
      for (int e = 0; e < K; ++e) o[e] = (v[e] - mean) * rstd * wr[e] + br[e];
      put_row(o, yr + i);
    });
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
  __shared__ float red[LOOP_THREADS / 64];
  for (long long row = blockIdx.x; row < s.outer; row += gridDim.x) {
    const T *xr = x + row * s.xo, *gr = dy + row * s.n;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float a1 = 0.f, a2 = 0.f;
    row_walk(xr, gr, s.n, [&](long long i, auto& v, auto& d) __attribute__((always_inline)) {
      constexpr int K = sizeof(v) / sizeof(float);
      float wr[K];
      load_params<K>(wr, w, s.pbf, i, 1.f);
#pragma unroll
      for (int e = 0; e < K; ++e) {
        a1 += d[e] * wr[e];
        a2 += d[e] * wr[e] * ((v[e] - mean) * rstd);
      }
    });
    const float c1 = loop_sum<LOOP_THREADS>(a1, red) * s.inv_n, c2 = loop_sum<LOOP_THREADS>(a2, red) * s.inv_n;
    row_walk(xr, gr, s.n, [&](long long i, auto& v, auto& d) __attribute__((always_inline)) {
      constexpr int K = sizeof(v) / sizeof(float);
      float wr[K], o[K];
      load_params<K>(wr, w, s.pbf, i, 1.f);
#pragma unroll
      for (int e = 0; e < K; ++e) o[e] = rstd * (d[e] * wr[e] - c1 - (v[e] - mean) * rstd * c2);
      put_row(o, dx + row * s.n + i);
    });
  }
}

// partial dw, db of slice blockIdx.y of the rows: a vector of columns a lane, the block's sixteen waves every sixteenth row
constexpr int DW_WAVES = LOOP_THREADS / 64;
template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_row_loop_dw(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd,
                                                               float* __restrict__ part, int slices) {
  constexpr int N = RtgVec<T>::N;
  __shared__ float red[DW_WAVES][64 * N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (long long c = (long long)blockIdx.x * 64 * N; c < s.n; c += (long long)gridDim.x * 64 * N) {
    const long long i = c + lane * N, at = i < s.n - N ? i : s.n - N;                   // (n >= N: ln_tiny has the rest)
    float aw[N], ab[N];
#pragma unroll
    for (int e = 0; e < N; ++e) aw[e] = ab[e] = 0.f;
    for (long long row = blockIdx.y * DW_WAVES + wave; row < s.outer; row += (long long)DW_WAVES * slices) {
      RtgVec<T> xv, gv;
      xv.load(x + row * s.xo + at);
      gv.load(dy + row * s.n + at);
      const float m = mean[row], r = rstd[row];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        aw[e] += gv.get(e) * ((xv.get(e) - m) * r);
        ab[e] += gv.get(e);
      }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < N; ++e) red[wave][lane * N + e] = which ? ab[e] : aw[e];
      __syncthreads();
      for (int j = threadIdx.x; j < 64 * N; j += LOOP_THREADS) {
        const long long first = c + j / N * N, col = first < s.n - N ? first : s.n - N;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < DW_WAVES; ++k) v += red[k][j];
        if (j % N >= first - col) part[((long long)blockIdx.y * 2 + which) * s.n + col + j % N] = v;
      }
    }
  }
}

// rows of less than a vector (fewer than 4 floats, than 8 bf16 values): a thread a row
constexpr int TINY_THREADS = 256, TINY_MOST = 7;
template <class T>
__global__ __launch_bounds__(TINY_THREADS) void ln_tiny_fwd(LnShape s, const T* __restrict__ x, const void* __restrict__ w,
                                                            const void* __restrict__ b, T* __restrict__ y, float* __restrict__ mean_out,
                                                            float* __restrict__ rstd_out) {
  const int n = (int)s.n;
  for (long long row = (long long)blockIdx.x * TINY_THREADS + threadIdx.x; row < s.outer; row += (long long)gridDim.x * TINY_THREADS) {
    float v[TINY_MOST], sum = 0.f, sq = 0.f;
#pragma unroll
    for (int e = 0; e < TINY_MOST; ++e) {
      v[e] = e < n ? rtg_up(x[row * s.xo + e]) : 0.f;
      sum += v[e];
    }
    const float mean = mean_of(sum, s);
#pragma unroll
    for (int e = 0; e < TINY_MOST; ++e) sq += e < n ? (v[e] - mean) * (v[e] - mean) : 0.f;
    const float rstd = rstd_of(sq, s);
#pragma unroll
    for (int e = 0; e < TINY_MOST; ++e)
      if (e < n) rtg_down((v[e] - mean) * rstd * param_at(w, s.pbf, e, 1.f) + param_at(b, s.pbf, e, 0.f), y[row * n + e]);
    if (mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

template <class T>
__global__ __launch_bounds__(TINY_THREADS) void ln_tiny_bwd(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                            const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                            const void* __restrict__ w, T* __restrict__ dx, float* __restrict__ part) {
  __shared__ float red[TINY_THREADS / 64][2 * TINY_MOST];
  const int n = (int)s.n;
  float aw[TINY_MOST], ab[TINY_MOST], wr[TINY_MOST];
#pragma unroll
  for (int e = 0; e < TINY_MOST; ++e) {
    aw[e] = ab[e] = 0.f;
    wr[e] = e < n ? param_at(w, s.pbf, e, 1.f) : 0.f;
  }
  for (long long row = (long long)blockIdx.x * TINY_THREADS + threadIdx.x; row < s.outer; row += (long long)gridDim.x * TINY_THREADS) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    float d[TINY_MOST], h[TINY_MOST], a1 = 0.f, a2 = 0.f;
#pragma unroll
    for (int e = 0; e < TINY_MOST; ++e) {
      d[e] = e < n ? rtg_up(dy[row * n + e]) : 0.f;
      h[e] = e < n ? (rtg_up(x[row * s.xo + e]) - mean) * rstd : 0.f;
      aw[e] += d[e] * h[e];
      ab[e] += d[e];
      a1 += d[e] * wr[e];
      a2 += d[e] * wr[e] * h[e];
    }
    if (!dx) continue;
    const float c1 = a1 * s.inv_n, c2 = a2 * s.inv_n;
#pragma unroll
    for (int e = 0; e < TINY_MOST; ++e)
      if (e < n) rtg_down(rstd * (d[e] * wr[e] - c1 - h[e] * c2), dx[row * n + e]);
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < TINY_MOST; ++e) {
    const float a = rtg_group_sum<64>(aw[e]), b = rtg_group_sum<64>(ab[e]);
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6][e] = a;
      red[threadIdx.x >> 6][TINY_MOST + e] = b;
    }
  }
  __syncthreads();
  const int which = threadIdx.x / 8, e = threadIdx.x % 8;
  if (which < 2 && e < n) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < TINY_THREADS / 64; ++k) v += red[k][which * TINY_MOST + e];
    part[((long long)blockIdx.x * 2 + which) * n + e] = v;
  }
}

// the sum over a block's waves of `v` at each lane, in every wave
__device__ __forceinline__ float wave_column_sum(float v, float (&red)[LOOP_THREADS / 64][64]) {
  const int lane = threadIdx.x & 63;
  __syncthreads();
  red[threadIdx.x >> 6][lane] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < LOOP_THREADS / 64; ++i) v += red[i][lane];
  return v;
}

// feature maps: a lane is a position, the waves share the channels
constexpr int MAP_WAVES = LOOP_THREADS / 64;
template <class T>
__global__ __launch_bounds__(LOOP_THREADS) void ln_map_loop_fwd(LnShape s, const T* __restrict__ x, const void* __restrict__ w,
                                                                const void* __restrict__ b, T* __restrict__ y,
                                                                float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float red[MAP_WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long tiles = (s.inner + 63) / 64;
  for (long long tile = blockIdx.x; tile < s.outer * tiles; tile += gridDim.x) {
    const long long o = tile / tiles, t = (tile - o * tiles) * 64 + lane;
    const bool in = t < s.inner;
    const T* xp = x + o * s.xo + t;
    float acc = 0.f;
    if (in)
#pragma unroll 4
      for (long long c = wave; c < s.n; c += MAP_WAVES) acc += rtg_up(xp[c * s.xn]);
    const float mean = mean_of(wave_column_sum(acc, red), s);
    acc = 0.f;
    if (in)
#pragma unroll 4
      for (long long c = wave; c < s.n; c += MAP_WAVES) {
        const float d = rtg_up(xp[c * s.xn]) - mean;
        acc += d * d;
      }
    const float rstd = rstd_of(wave_column_sum(acc, red), s);
    if (!in) continue;
    T* yp = y + o * s.n * s.inner + t;
#pragma unroll 4
    for (long long c = wave; c < s.n; c += MAP_WAVES)
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
  __shared__ float red[MAP_WAVES][64];
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
#pragma unroll 4
      for (long long c = wave; c < s.n; c += MAP_WAVES) {
        const float g = rtg_up(gp[c * s.inner]) * param_at(w, s.pbf, c, 1.f);
        a1 += g;
        a2 += g * ((rtg_up(xp[c * s.xn]) - mean) * rstd);
      }
    }
    const float c1 = wave_column_sum(a1, red) * s.inv_n, c2 = wave_column_sum(a2, red) * s.inv_n;
    if (!in) continue;
    T* dp = dx + o * s.n * s.inner + t;
#pragma unroll 4
    for (long long c = wave; c < s.n; c += MAP_WAVES) {
      const float g = rtg_up(gp[c * s.inner]) * param_at(w, s.pbf, c, 1.f);
      rtg_down(rstd * (g - c1 - (rtg_up(xp[c * s.xn]) - mean) * rstd * c2), dp[c * s.inner]);
    }
  }
}

// partial dw, db of one channel (blockIdx.x) over slice blockIdx.y of the clips: adjacent positions in adjacent threads
template <class T>
__global__ __launch_bounds__(TINY_THREADS) void ln_map_loop_dw(LnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd,
                                                               float* __restrict__ part, int slices) {
  __shared__ float red[TINY_THREADS / 64];
  const long long total = s.outer * s.inner;
  for (long long c = blockIdx.x; c < s.n; c += gridDim.x) {
    float aw = 0.f, ab = 0.f;
#pragma unroll 4
    for (long long p = (long long)blockIdx.y * TINY_THREADS + threadIdx.x; p < total; p += (long long)slices * TINY_THREADS) {
      const long long o = p / s.inner, t = p - o * s.inner;
      const float g = rtg_up(dy[(o * s.n + c) * s.inner + t]);
      aw += g * ((rtg_up(x[o * s.xo + c * s.xn + t]) - mean[p]) * rstd[p]);
      ab += g;
    }
    aw = loop_sum<TINY_THREADS>(aw, red);
    ab = loop_sum<TINY_THREADS>(ab, red);
    if (threadIdx.x == 0) {
      part[((long long)blockIdx.y * 2) * s.n + c] = aw;
      part[((long long)blockIdx.y * 2 + 1) * s.n + c] = ab;
    }
  }
}

// dw, db = the sums of their `slices` partials [slice][dw | db][n], each in the order of the slices: 32 columns a block, a
// column's slices over 32 threads (so that the reads of a column are in flight together), then a fixed tree: 256 partials of 2048
// columns in 4 us
__global__ __launch_bounds__(FIN_COLS* FIN_ROWS) void ln_finish(const float* __restrict__ part, int slices, long long n,
                                                                void* __restrict__ dw, void* __restrict__ db, int pbf) {
  __shared__ float red[FIN_ROWS][FIN_COLS + 1];
  void* const out = blockIdx.y ? db : dw;
  if (!out) return;                                        // (the whole block)
  const int col = threadIdx.x % FIN_COLS, r = threadIdx.x / FIN_COLS;
  for (long long c = (long long)blockIdx.x * FIN_COLS; c < n; c += (long long)gridDim.x * FIN_COLS) {
    const long long i = c + col;
    float acc = 0.f;
    if (i < n) {
      const float* p = part + (long long)blockIdx.y * n + i;
      int q = r;
      for (; q + 7 * FIN_ROWS < slices; q += 8 * FIN_ROWS) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = p[(long long)(q + k * FIN_ROWS) * 2 * n];
#pragma unroll
        for (int k = 0; k < 8; ++k) acc += v[k];
      }
      for (; q < slices; q += FIN_ROWS) acc += p[(long long)q * 2 * n];
    }
    red[r][col] = acc;
    __syncthreads();
#pragma unroll
    for (int h = FIN_ROWS / 2; h > 0; h >>= 1) {
      if (r < h) red[r][col] += red[r + h][col];
      __syncthreads();
    }
    if (r == 0 && i < n) put_param(out, pbf, i, red[0][col]);   // (red[0] is these threads' own until the next barrier)
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
inline long long lmin(long long a, long long b) { return a < b ? a : b; }

// A launch holds blocks x threads in 32 bits (more are cut off without an error), so at most 2^21 blocks of up to 1024 threads, a
// multiple of 8 (xcd_order).  The kernels with a block for each of something stride over more of it; ln_map_fwd, a tile a team, is
// launched again for the rest
constexpr int MOST_BLOCKS = 1 << 21;

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

// tensors: how many of the problem's size a kernel reads
LnShape shape_of(const RtgLayerNormDesc* d, int tensors) {
  return LnShape{d->outer, d->n, d->inner, d->x_outer, d->x_n, (float)d->n, (float)(1.0 / (double)d->n), d->eps, d->param_bf16 != 0,
                 d->outer * d->n * d->inner >= CACHED / ((d->bf16 ? 2 : 4) * tensors)};
}

bool is_rows(const RtgLayerNormDesc* d) { return d->inner == 1; }

// What serves a problem: the smallest register tile that holds the normalised axis, else the kernels for any size.  `tile` is
// the tile's number in the dispatch below, `blocks` the grid, in the backward also the number of partial dw / db.
struct Plan { int tile; int blocks; };
constexpr int LOOPS = -1, TINY = -2;

// Rows: threads per row, 16-byte vectors per thread, threads per block.  Over 13 widths from 64 to 16384 and row counts from 1 to
// 65536 these tiles are within 5 % of the best of 20 (forward) and 40 (backward); what they weigh: a wave's rows need no
// barrier (up to two vectors a thread), a block's row two; the backward holds sixteen elements a thread at most (the weight, dw
// and db take a register each).  The shortest rows have eight lanes whatever their length: of five floats two are busy (1000000
// rows of them 18.8 us forward, 35.6 backward).  Forward, as many blocks as fit up to 64 MB of rows (8192 x 2048 bf16, side by
// side, 14.2 us, with half of them 15.6, and 13.6 .. 16.0 from program to program; 4096 x 1024 floats 7.8 and 8.5; not of 1024
// threads: 2048 x 16384 bf16 28.7 and 26.9), half of them beyond: each walks its
// rows with the next in flight, and fewer rows of HBM are open at a time (65536 x 1024 floats 81 us, with all of them 83, with a
// quarter 110; 16384 x 4096 bf16 45.8, 48.6, 50.2).
struct RowTile { int tpr, vpt, blk; };
constexpr int ROW_TILES = 10;
constexpr RowTile FWD_TILES[ROW_TILES] = {{8, 1, 256},   {16, 1, 256},  {32, 1, 256},  {64, 1, 256},   {64, 2, 256},
                                          {256, 1, 256}, {256, 2, 256}, {512, 2, 512}, {1024, 2, 1024}, {1024, 4, 1024}};
constexpr RowTile BWD_F32[ROW_TILES] = {{8, 1, 512},    {16, 1, 512},  {32, 1, 512},  {64, 1, 512},    {64, 2, 512},
                                        {256, 1, 1024}, {256, 2, 512}, {512, 2, 512}, {1024, 2, 1024}, {1024, 3, 1024}};
constexpr RowTile BWD_BF16[ROW_TILES] = {{8, 1, 512},   {16, 1, 512},  {32, 1, 512},  {64, 1, 512},    {64, 2, 512},
                                         {256, 1, 512}, {256, 2, 512}, {512, 2, 512}, {1024, 2, 1024}, {1024, 2, 1024}};

int row_tile(const RowTile* tiles, long long n, int bf16) {
  const int vec = bf16 ? 8 : 4;
  if (n < vec) return TINY;
  const long long nv = (n + vec - 1) / vec;
  for (int i = 0; i < ROW_TILES; ++i)
    if (nv <= tiles[i].tpr * tiles[i].vpt) return i;
  return LOOPS;
}

// Maps: position lanes, waves that share the channels, channels a lane, as one number (the dispatch's label).  Over 12 channel
// counts from 8 to 1024 and 7 sizes of map each, both types, the rules below are 2 % (forward) and 3 % (backward) behind the best
// of all 38 tiles; what they weigh:
//   - the channels are just covered: 32 channels by 8 x 4 lanes' worth 14.9 us of a 67 MB map, by twice as many 17.3;
//   - a wide tile (a line of 128 bytes of each channel, 16 channels a lane: few waves meet for a sum) where its waves fill the
//     chip twice: 128 channels x 65536 positions 13.5 us against 17.4 with four channels a lane and four waves; with 1024
//     positions it is the other way round, 4.6 against 3.6: more waves, fewer loads each;
//   - two position lanes where a clip has no more than two vectors of positions (512 channels x 8: 3.7 us against 4.2).
//   - single elements in the place of vectors where a clip has fewer positions than a vector.
constexpr int map_key(int lp, int w, int cpt, bool one = false) { return (one ? 1000000 : 0) + lp * 10000 + w * 100 + cpt; }
#define LN_MAP_FWD(X) \
  X(16, 1, 2) X(16, 1, 4) X(8, 1, 4) X(8, 2, 4) X(8, 4, 4) X(4, 4, 4) X(4, 8, 4) X(2, 1, 4) X(2, 2, 4) X(2, 4, 4) X(2, 8, 4) \
  X(8, 1, 8) X(8, 1, 16) X(8, 2, 16) X(8, 4, 16) X(8, 8, 16) X(4, 16, 8)
#define LN_MAP_BWD(X) \
  X(16, 1, 2) X(16, 1, 4) X(8, 1, 4) X(8, 2, 4) X(8, 4, 4) X(8, 8, 4) X(4, 4, 4) X(4, 8, 4) X(2, 1, 4) X(2, 2, 4) X(2, 4, 4) X(2, 8, 4) \
  X(8, 2, 8) X(8, 8, 8) X(4, 8, 8) X(2, 16, 4)
#define LN_MAP_ONE(X) X(8, 1, 4) X(8, 4, 4) X(8, 8, 8) X(8, 8, 16)

#define LN_MAP(LP, W, CPT) LN_MAP_CASE(RtgVec<T>, false, LP, W, CPT)
#define LN_MAP1(LP, W, CPT) LN_MAP_CASE(RtgOne<T>, true, LP, W, CPT)

bool map_one(const RtgLayerNormDesc* d) { return d->inner < (d->bf16 ? 8 : 4); }
long long map_tiles(const RtgLayerNormDesc* d, int lp) {
  const long long pos = lp * (map_one(d) ? 1 : d->bf16 ? 8 : 4);
  return d->outer * ((d->inner + pos - 1) / pos);
}
// (two vectors of positions a clip at most)
int map_short_key(long long n) {
  return n <= 128 ? map_key(2, 1, 4) : n <= 256 ? map_key(2, 2, 4) : n <= 512 ? map_key(2, 4, 4) : map_key(2, 8, 4);
}
int map_one_key(long long n) {
  return n <= 32 ? map_key(8, 1, 4, true) : n <= 128 ? map_key(8, 4, 4, true) : n <= 512 ? map_key(8, 8, 8, true) : map_key(8, 8, 16, true);
}
// two of a wide tile's waves for every SIMD (256 CUs of four)
bool map_wide(const RtgLayerNormDesc* d, int lp, int w) { return map_tiles(d, lp) * w >= 2048; }

int map_fwd(const RtgLayerNormDesc* d) {
  const long long n = d->n;
  if (map_one(d)) return map_one_key(n);
  if (d->inner <= (d->bf16 ? 16 : 8) && n <= 1024) return map_short_key(n);
  if (n <= 8) return map_key(16, 1, 2);
  if (n <= 16) return map_key(16, 1, 4);
  if (n <= 32) return map_key(8, 1, 4);
  if (n <= 64) return map_wide(d, 8, 1) ? map_key(8, 1, 8) : map_key(8, 2, 4);
  if (n <= 128) return map_wide(d, 8, 1) ? map_key(8, 1, 16) : map_key(8, 4, 4);
  if (n <= 256) return map_wide(d, 8, 2) ? map_key(8, 2, 16) : map_key(4, 4, 4);
  if (n <= 512) return map_wide(d, 8, 4) ? map_key(8, 4, 16) : map_tiles(d, 8) >= 64 ? map_key(4, 8, 4) : map_key(2, 4, 4);
  if (n <= 1024) return map_wide(d, 8, 8) ? map_key(8, 8, 16) : map_key(2, 8, 4);
  return map_key(4, 16, 8);
}

int map_bwd(const RtgLayerNormDesc* d) {
  const long long n = d->n;
  if (map_one(d)) return map_one_key(n);
  if (d->inner <= (d->bf16 ? 16 : 8) && n <= 1024) return map_short_key(n);
  if (n <= 8) return map_key(16, 1, 2);
  if (n <= 16) return map_key(16, 1, 4);
  if (n <= 32) return map_key(8, 1, 4);
  if (n <= 64) return map_key(8, 2, 4);
  if (n <= 128) return map_wide(d, 8, 1) ? map_key(8, 2, 8) : map_key(8, 4, 4);
  if (n <= 256) return map_wide(d, 8, 8) ? map_key(8, 8, 4) : map_key(4, 4, 4);
  if (n <= 512) return map_wide(d, 8, 4) ? map_key(8, 8, 8) : map_key(4, 8, 4);
  if (n <= 1024) return map_wide(d, 4, 8) ? map_key(4, 8, 8) : map_key(2, 8, 4);
  return map_key(2, 16, 4);
}

// blocks that give each team one tile; 0: no register tile holds the problem (or a lane's offset in a tile would pass 32 bits)
long long map_blocks(const RtgLayerNormDesc* d, int key) {
  const int lp = key / 10000 % 100, w = key / 100 % 100, cpt = key % 100;
  if (d->n > 64 / lp * w * cpt || d->inner >= 1 << 24 || d->x_n >= 1 << 24) return 0;
  const long long tiles = map_tiles(d, lp), teams = map_teams(w);
  return tiles >= 1ll << 30 ? 0 : (tiles + teams - 1) / teams;
}

// blocks for `items` tiles of work, at most `cap` of them with as even a share as can be
int even_blocks(long long items, long long cap) {
  const long long rounds = (items + cap - 1) / cap;
  return (int)((items + rounds - 1) / rounds);
}

Plan plan_fwd(const RtgLayerNormDesc* d) {
  if (is_rows(d)) {
    const int i = row_tile(FWD_TILES, d->n, d->bf16);
    if (i == LOOPS) return {LOOPS, (int)lmin(d->outer, 1 << 20)};
    if (i == TINY) return {TINY, even_blocks((d->outer + TINY_THREADS - 1) / TINY_THREADS, 2048)};
    const int groups = FWD_TILES[i].blk / FWD_TILES[i].tpr;
    const bool all = d->outer * d->n * (d->bf16 ? 2 : 4) <= 64ll << 20 && FWD_TILES[i].blk < 1024;
    const int threads = all ? 2048 : 1024;                 // a CU
    return {i, even_blocks((d->outer + groups - 1) / groups, 256 * (threads / FWD_TILES[i].blk))};
  }
  const int key = map_fwd(d);
  const long long blocks = map_blocks(d, key);
  if (blocks == 0) return {LOOPS, (int)lmin(d->outer * ((d->inner + 63) / 64), 1 << 20)};
  return {key, ((int)blocks + 7) / 8 * 8};
}

Plan plan_bwd(const RtgLayerNormDesc* d) {
  if (is_rows(d)) {
    const RowTile* tiles = d->bf16 ? BWD_BF16 : BWD_F32;
    const int i = row_tile(tiles, d->n, d->bf16);
    if (i == TINY) return {TINY, even_blocks((d->outer + TINY_THREADS - 1) / TINY_THREADS, 512)};
    if (i == LOOPS) {
      const long long wide = 64 * (d->bf16 ? 8 : 4), cols = (d->n + wide - 1) / wide;
      const long long s = lmin((d->outer + 2 * DW_WAVES - 1) / (2 * DW_WAVES), (512 + cols - 1) / cols);
      return {LOOPS, (int)(s < 1 ? 1 : s)};
    }
    // 256 blocks: two partials a CU would be more to add than the second block gains.  One block alone writes dw and db
    // itself; it is worth that for a few rounds of rows (16 x 512: 4.4 us, in two blocks and ln_finish 5.7).
    const int groups = tiles[i].blk / tiles[i].tpr;
    const long long rounds = (d->outer + groups - 1) / groups;
    // A block that holds one long row at a time walks two at least, or there is as much of the partials as of the rows
    // (256 x 8192 floats 16.6 -> 14.7 us).
    const long long cap = groups == 1 ? lmin(256, (rounds + 1) / 2) : 256;
    return {i, rounds <= (tiles[i].tpr <= 64 ? 4 : 1) ? 1 : even_blocks(rounds, cap)};
  }
  const int key = map_bwd(d);
  const long long blocks = map_blocks(d, key);
  if (blocks > 0) return {key, (even_blocks(blocks, key / 100 % 100 * (key % 100) >= 64 ? 256 : 512) + 7) / 8 * 8};
  const long long s = lmin((d->outer * d->inner + 1023) / 1024, (2048 + d->n - 1) / d->n);
  return {LOOPS, (int)(s < 1 ? 1 : lmin(s, 1024))};
}

dim3 finish_grid(long long n) { return dim3((unsigned)lmin(rtg_ceil_div(n, FIN_COLS), MOST_BLOCKS), 2); }

template <class T>
int forward(const RtgLayerNormDesc* d, const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, hipStream_t st) {
  const LnShape s = shape_of(d, 1);
  const T* xt = reinterpret_cast<const T*>(x);
  T* yt = reinterpret_cast<T*>(y);
  const Plan p = plan_fwd(d);
#define LN_ROW(I)                                                                                                            \
  case I: {                                                                                                                  \
    constexpr RowTile R = FWD_TILES[I];                                                                                      \
    constexpr int AHEAD = R.tpr * R.vpt < 4096;                                                                              \
    if (s.once)                                                                                                              \
      RTG_KLAUNCH((ln_row_fwd<T, R.tpr, R.vpt, R.blk, AHEAD, true>), dim3(p.blocks), dim3(R.blk), 0, st, s, xt, w, b, yt, mean, rstd); \
    else                                                                                                                     \
      RTG_KLAUNCH((ln_row_fwd<T, R.tpr, R.vpt, R.blk, AHEAD, false>), dim3(p.blocks), dim3(R.blk), 0, st, s, xt, w, b, yt, mean, rstd); \
    return rtg_launch_status();                                                                                              \
  }
#define LN_MAP_CASE(VEC, ONE, LP, W, CPT)                                                                                    \
  case map_key(LP, W, CPT, ONE):                                                                                             \
    for (int at = 0; at < p.blocks; at += MOST_BLOCKS) {                                                                       \
      RTG_KLAUNCH((ln_map_fwd<VEC, LP, W, CPT>), dim3((unsigned)lmin(p.blocks - at, MOST_BLOCKS)), dim3(map_block(W)), 0, st, s, xt, w, b, \
                  yt, mean, rstd, (unsigned)at);                                                                             \
      const int rc = rtg_launch_status();                                                                                    \
      if (rc != RTG_OK) return rc;                                                                                           \
    }                                                                                                                        \
    return RTG_OK;
  if (is_rows(d)) {
    switch (p.tile) {
      LN_ROW(0) LN_ROW(1) LN_ROW(2) LN_ROW(3) LN_ROW(4) LN_ROW(5) LN_ROW(6) LN_ROW(7) LN_ROW(8) LN_ROW(9)
    }
    if (p.tile == TINY) RTG_KLAUNCH(ln_tiny_fwd<T>, dim3(p.blocks), dim3(TINY_THREADS), 0, st, s, xt, w, b, yt, mean, rstd);
    else RTG_KLAUNCH(ln_row_loop_fwd<T>, dim3(p.blocks), dim3(LOOP_THREADS), 0, st, s, xt, w, b, yt, mean, rstd);
  } else {
    switch (p.tile) {
      LN_MAP_FWD(LN_MAP)
      LN_MAP_ONE(LN_MAP1)
    }
    RTG_KLAUNCH(ln_map_loop_fwd<T>, dim3(p.blocks), dim3(LOOP_THREADS), 0, st, s, xt, w, b, yt, mean, rstd);
  }
#undef LN_ROW
#undef LN_MAP_CASE
  return rtg_launch_status();
}

template <class T>
int backward(const RtgLayerNormDesc* d, const void* dy, const void* x, const float* mean, const float* rstd, const void* w, void* dx,
             void* dw, void* db, float* ws, hipStream_t st) {
  const LnShape s = shape_of(d, 2);
  const T *xt = reinterpret_cast<const T*>(x), *gt = reinterpret_cast<const T*>(dy);
  T* dt = reinterpret_cast<T*>(dx);
  const bool params = dw || db;
  if (!dx && !params) return RTG_OK;
  float* const part = params ? ws : nullptr;
  const Plan p = plan_bwd(d);
#define LN_ROW(I)                                                                                                            \
  case I: {                                                                                                                  \
    constexpr RowTile R = sizeof(T) == 2 ? BWD_BF16[I] : BWD_F32[I];                                                         \
    constexpr int AHEAD = R.tpr < 1024;                                                                                      \
    if (s.once)                                                                                                              \
      RTG_KLAUNCH((ln_row_bwd<T, R.tpr, R.vpt, R.blk, AHEAD, true>), dim3(p.blocks), dim3(R.blk), 0, st, s, gt, xt, mean, rstd, w, dt, \
                  part, dw, db);                                                                                             \
    else                                                                                                                     \
      RTG_KLAUNCH((ln_row_bwd<T, R.tpr, R.vpt, R.blk, AHEAD, false>), dim3(p.blocks), dim3(R.blk), 0, st, s, gt, xt, mean, rstd, w, dt, \
                  part, dw, db);                                                                                             \
    break;                                                                                                                   \
  }
#define LN_MAP_CASE(VEC, ONE, LP, W, CPT)                                                                                    \
  case map_key(LP, W, CPT, ONE):                                                                                             \
    RTG_KLAUNCH((ln_map_bwd<VEC, LP, W, CPT>), dim3(p.blocks), dim3(map_block(W)), 0, st, s, gt, xt, mean, rstd, w, dt, part);  \
    break;
  if (p.tile == TINY) {
    RTG_KLAUNCH(ln_tiny_bwd<T>, dim3(p.blocks), dim3(TINY_THREADS), 0, st, s, gt, xt, mean, rstd, w, dt, part);
  } else if (is_rows(d) && p.tile != LOOPS) {
    switch (p.tile) {
      LN_ROW(0) LN_ROW(1) LN_ROW(2) LN_ROW(3) LN_ROW(4) LN_ROW(5) LN_ROW(6) LN_ROW(7) LN_ROW(8) LN_ROW(9)
    }
  } else if (is_rows(d)) {
    if (dx) {
      RTG_KLAUNCH(ln_row_loop_dx<T>, dim3((unsigned)lmin(d->outer, 1 << 20)), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, w, dt);
      const int rc = rtg_launch_status();
      if (rc != RTG_OK) return rc;
    }
    if (params)
      RTG_KLAUNCH(ln_row_loop_dw<T>, dim3((unsigned)lmin(rtg_ceil_div(d->n, 64 * RtgVec<T>::N), MOST_BLOCKS / p.blocks), p.blocks), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean,
                  rstd, part, p.blocks);
  } else if (p.tile != LOOPS) {
    switch (p.tile) {
      LN_MAP_BWD(LN_MAP)
      LN_MAP_ONE(LN_MAP1)
    }
  } else {
    if (dx) {
      const long long tiles = d->outer * ((d->inner + 63) / 64);
      RTG_KLAUNCH(ln_map_loop_dx<T>, dim3((unsigned)lmin(tiles, 1 << 20)), dim3(LOOP_THREADS), 0, st, s, gt, xt, mean, rstd, w, dt);
      const int rc = rtg_launch_status();
      if (rc != RTG_OK) return rc;
    }
    if (params)
      RTG_KLAUNCH(ln_map_loop_dw<T>, dim3((unsigned)lmin(d->n, 1 << 20), p.blocks), dim3(TINY_THREADS), 0, st, s, gt, xt, mean, rstd, part,
                  p.blocks);
  }
#undef LN_ROW
#undef LN_MAP_CASE
  const int rc = rtg_launch_status();
  if (rc != RTG_OK || !params || (is_rows(d) && p.tile >= 0 && p.blocks == 1)) return rc;   // (one block: dw, db are written)
  RTG_KLAUNCH(ln_finish, finish_grid(d->n), dim3(FIN_COLS * FIN_ROWS), 0, st, (const float*)ws, p.blocks,
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
    RTG_KLAUNCH(ln_finish, finish_grid(d->n), dim3(FIN_COLS * FIN_ROWS), 0, (hipStream_t)stream,
                (const float*)nullptr, 0, d->n, dweight, dbias, d->param_bf16 != 0);
    return rtg_launch_status();
  }
  if (!dy || !x || !mean || !rstd || (params && !ws)) return RTG_ENULL;
  return d->bf16 ? backward<rtg_bf16>(d, dy, x, mean, rstd, weight, dx, dweight, dbias, ws, (hipStream_t)stream)
                 : backward<float>(d, dy, x, mean, rstd, weight, dx, dweight, dbias, ws, (hipStream_t)stream);
}

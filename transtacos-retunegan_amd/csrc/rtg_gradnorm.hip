// rtg_gradnorm.hip — the norm over many gradient tensors, clipping by it, and the AdamW update that reads clipped gradients
// (see include/rtg.h, rtg_grad_norm / rtg_grad_clip / rtg_adamw_clipped).
//
//   norm = sqrt(sum_t sum_i g_t[i]^2)  or  max |g|;   factor = min(1, max_norm / (norm + 1e-6))
//
// One multiply-add per element of 2 or 4 bytes: bound by HBM (and, for a small model, by the launches).  The tensors are cut
// into chunks of one size, whatever their number: 172 tensors of a generator are one launch.  A workgroup takes every so many-th
// chunk, so that all of them together walk the list from its start to its end (adjacent pages of HBM at any one time: 134 M
// floats clipped in 278 us, with one long chunk a workgroup 296).  A workgroup's sum is a double: the square of any float is a normal double, so nothing overflows or vanishes, and the result does not depend
// on how a list is cut into tensors beyond the last bits of a double.
#include "rtg_vec.h"
#include <algorithm>
#include <memory>
#include <new>

namespace {

constexpr int TABLE = 192;            // tensors per launch: the table travels in the kernel's arguments (3.9 KB of 4)
constexpr int JOBS = 32;              // AdamW buffers per launch
constexpr int THREADS = 256;
constexpr int REDUCE = 1024;

struct GradTable {
  void* p[TABLE];
  long long n[TABLE];
  int first[TABLE];                   // first chunk of tensor i in this launch (increasing; empty tensors have none)
  unsigned bf16[TABLE / 32];
  int count, chunks;
  long long chunk;                    // bytes of a chunk, a multiple of 4096
};

// the table's entry that workgroup b works on: the last one with first <= b.  Every lane compares its own entries (one round
// of loads in flight together; a binary search is eight dependent ones)
__device__ __forceinline__ int entry_of(const int* first, int count, int b) {
  int found = 0;
#pragma unroll
  for (int k = 0; k < (TABLE + 63) / 64; ++k) {
    const int i = k * 64 + (threadIdx.x & 63);
    found += __popcll(__ballot(i < count && first[i] <= b));
  }
  return __builtin_amdgcn_readfirstlane(found) - 1;
}

template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
  if constexpr (KIND == RTG_NORM_L2) return a + b;
  return (b > a || b != b) ? b : a;                      // (a NaN stays: nothing compares greater)
}
template <int KIND>
__device__ __forceinline__ double take(double acc, float v) {
  if constexpr (KIND == RTG_NORM_L2) return fma((double)v, (double)v, acc);
  return join<KIND>(acc, (double)fabsf(v));
}

// over the N threads of a block, result in every thread; `red`: N / 64 doubles of LDS
template <int KIND, int N>
__device__ __forceinline__ double block_join(double v, double* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = join<KIND>(v, __shfl_xor(v, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < N / 64; ++i) v = join<KIND>(v, red[i]);
  return v;
}

// the partials of all chunks, in an order their number decides; result in every thread
template <int KIND, int N>
__device__ __forceinline__ double all_partials(const double* __restrict__ part, int n, double* red) {
  double acc = 0.0;
  int i = threadIdx.x;
  for (; i + 7 * N < n; i += 8 * N) {                    // (eight loads in flight: one after the other they are microseconds)
    double v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = part[i + k * N];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc = join<KIND>(acc, v[k]);
  }
  for (; i < n; i += N) acc = join<KIND>(acc, part[i]);
  return block_join<KIND, N>(acc, red);
}

template <int KIND>
__device__ __forceinline__ double norm_of(double joined) { return KIND == RTG_NORM_L2 ? sqrt(joined) : joined; }

// min(1, max_norm / (norm + 1e-6)) of the norm in 64 bits: 0 for an infinite norm, NaN for a NaN
__device__ __forceinline__ float clip_factor(double norm, double max_norm) {
  const double f = max_norm / (norm + 1e-6);
  return f < 1.0 || f != f ? (float)f : 1.f;
}

// elements in front of the first whole word (a bf16 tensor may start in the middle of one: its vectors would be 4.7 TB/s,
// those that start with a word 5.7, whatever the line)
template <class T>
__device__ __forceinline__ int odd_head(const T* p, long long n) {
  return sizeof(T) == 2 && n > 0 && (reinterpret_cast<uintptr_t>(p) & 2) ? 1 : 0;
}

template <class T, int KIND, bool ONCE>
__device__ __forceinline__ double chunk_sum(const T* __restrict__ p, long long n) {
  constexpr int N = RtgVec<T>::N;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  const int head = odd_head(p, n);
  if (head && threadIdx.x == 0) acc[3] = take<KIND>(acc[3], rtg_up(*p));
  p += head;
  n -= head;
  const long long nv = n / N;
  long long i = threadIdx.x;
  for (; i + 3 * THREADS < nv; i += 4 * THREADS) {
    RtgVec<T> v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) rtg_load<ONCE>(v[k], p + (i + k * THREADS) * N);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) acc[k] = take<KIND>(acc[k], v[k].get(e));
  }
  for (; i < nv; i += THREADS) {
    RtgVec<T> v;
    rtg_load<ONCE>(v, p + i * N);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[0] = take<KIND>(acc[0], v.get(e));
  }
  if (nv * N + threadIdx.x < n) acc[1] = take<KIND>(acc[1], rtg_up(p[nv * N + threadIdx.x]));
  return join<KIND>(join<KIND>(acc[0], acc[1]), join<KIND>(acc[2], acc[3]));
}

// chunk b: [lo, lo + n) of entry i
struct Piece { int i; long long lo, n; bool bf; };
__device__ __forceinline__ Piece piece_of(const GradTable& t, int b) {
  Piece r;
  r.i = entry_of(t.first, t.count, b);
  r.bf = (t.bf16[r.i >> 5] >> (r.i & 31)) & 1;
  const long long size = t.chunk >> (r.bf ? 1 : 2);
  r.lo = (long long)(b - t.first[r.i]) * size;
  const long long left = t.n[r.i] - r.lo;
  r.n = left < size ? left : size;
  return r;
}

// Who reads a tensor again, and from where: a list of up to CACHED bytes is still in the memory-side cache (256 MB) when the
// scaling or the update comes, so its norm leaves it there and the scaling, its last reader, makes no room for what it reads and
// writes (27 M floats clipped in 58 us; with plain accesses 8 more, with both passes that way 12: the second then reads HBM).  Of
// a longer list nothing is left by then: its norm reads past the caches (1 GB of bf16 184 us, 5.8 TB/s, with plain reads 17
// more; clipped 591 and 55 more).
constexpr long long CACHED = 256ll << 20;

template <int KIND, bool ONCE>
__global__ __launch_bounds__(THREADS) void grad_partial(const GradTable t, double* __restrict__ part) {
  __shared__ double red[THREADS / 64];
  double acc = 0.0;
  for (int b = blockIdx.x; b < t.chunks; b += gridDim.x) {
    const Piece c = piece_of(t, b);
    double sum;
    if (c.bf) sum = chunk_sum<rtg_bf16, KIND, ONCE>(reinterpret_cast<const rtg_bf16*>(t.p[c.i]) + c.lo, c.n);
    else sum = chunk_sum<float, KIND, ONCE>(reinterpret_cast<const float*>(t.p[c.i]) + c.lo, c.n);
    acc = join<KIND>(acc, sum);
  }
  acc = block_join<KIND, THREADS>(acc, red);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

template <int KIND>
__global__ __launch_bounds__(REDUCE) void grad_norm_finish(double* part, int n, float* __restrict__ out, int joined) {
  __shared__ double red[REDUCE / 64];
  const double acc = all_partials<KIND, REDUCE>(part, n, red);
  if (threadIdx.x != 0) return;
  *out = (float)norm_of<KIND>(acc);
  if (joined) part[0] = acc;                             // (behind the barriers of the sum: all have read it)
}

template <class T, bool ONCE>
__device__ __forceinline__ void chunk_scale(T* __restrict__ p, long long n, float f) {
  constexpr int N = RtgVec<T>::N;
  const int head = odd_head(p, n);
  if (head && threadIdx.x == 0) rtg_down(rtg_up(*p) * f, *p);
  p += head;
  n -= head;
  const long long nv = n / N;
  for (long long i = threadIdx.x; i < nv; i += THREADS) {
    RtgVec<T> v;
    float r[N];
    rtg_load<ONCE>(v, p + i * N);
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = v.get(e) * f;
    v.set(r);
    rtg_store<ONCE>(v, p + i * N);
  }
  if (nv * N + threadIdx.x < n) rtg_down(rtg_up(p[nv * N + threadIdx.x]) * f, p[nv * N + threadIdx.x]);
}

// scales the chunks whose sums it may have taken.  Up to JOIN_FIRST partials every workgroup joins them by itself (they sit in L2;
// a launch of one workgroup for it costs more: 2.7 M elements 13.1 us, with it 14.7); of more, the first one holds what that
// launch made of them (2 GB of floats within the limit 459 -> 426 us, 30000 tensors 1931 -> 1386)
constexpr int JOIN_FIRST = 4096;
template <int KIND, bool ONCE>
__global__ __launch_bounds__(THREADS) void grad_scale(const GradTable t, const double* __restrict__ part, int n_part, double max_norm,
                                                      float* __restrict__ out, int write_norm) {
  __shared__ double red[THREADS / 64];
  const double norm = norm_of<KIND>(all_partials<KIND, THREADS>(part, n_part, red));
  if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *out = (float)norm;
  const float f = clip_factor(norm, max_norm);
  if (f == 1.f) return;
  for (int b = blockIdx.x; b < t.chunks; b += gridDim.x) {
    const Piece c = piece_of(t, b);
    if (c.bf) chunk_scale<rtg_bf16, ONCE>(reinterpret_cast<rtg_bf16*>(t.p[c.i]) + c.lo, c.n, f);
    else chunk_scale<float, ONCE>(reinterpret_cast<float*>(t.p[c.i]) + c.lo, c.n, f);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// AdamW over flat buffers with clipped gradients: torch.optim.AdamW's order of operations (adamw_kernel, rtg_elem.hip)
// ---------------------------------------------------------------------------------------------------------------------
struct AdamTable {
  RtgAdamWJob job[JOBS];
  int first[JOBS];
  int count;
  long long chunk;                    // elements, a multiple of 1024
};
struct AdamScalars { float step_size, bc2s, scale, go; };        // go 0: the buffer is left alone
struct AdamRates { double max_norm, lr, b1, b2; float gscale; };

__device__ __forceinline__ double adam_norm(double joined, const AdamRates& r) { return sqrt(joined) * fabs((double)r.gscale); }
// step: the counter before this update
__device__ __forceinline__ AdamScalars adam_scalars(double norm, float step, bool flagged, const AdamRates& r) {
  const double t = (double)step + 1.0;
  AdamScalars s;
  s.step_size = (float)(r.lr / (1.0 - pow(r.b1, t)));
  s.bc2s = (float)sqrt(1.0 - pow(r.b2, t));
  s.scale = r.gscale * clip_factor(norm, r.max_norm);
  s.go = isfinite((float)norm) && !flagged ? 1.f : 0.f;   // (the norm as the caller sees it)
  return s;
}
__device__ __forceinline__ bool adam_flagged(const float* flag) { return flag && isnan(*flag); }

// Many partials or buffers: one workgroup between the norm and the update takes the factor and each buffer's bias corrections
// once, and advances the step counters behind the last reader of the old ones
__global__ __launch_bounds__(REDUCE) void adam_prepare(const AdamTable t, const double* __restrict__ part, int n_part, const AdamRates r,
                                                       AdamScalars* __restrict__ sc, float* __restrict__ norm_out, int write_norm) {
  __shared__ double red[REDUCE / 64];
  const double norm = adam_norm(all_partials<RTG_NORM_L2, REDUCE>(part, n_part, red), r);
  const int j = threadIdx.x;
  if (j == 0 && write_norm && norm_out) *norm_out = (float)norm;
  if (j >= t.count) return;
  const float step = t.job[j].step_state[0];
  const AdamScalars s = adam_scalars(norm, step, adam_flagged(t.job[j].loss_flag), r);
  sc[j] = s;
  if (s.go != 0.f) t.job[j].step_state[0] = step + 1.f;
}

// Few of them: the partial sums carry the counters and flags as they were (`held`), so that every workgroup of the update makes
// the scalars itself and one of them may advance the counter at once: two launches (2.7 M parameters 22.4 -> 21.2 us, 1000 parameters 8.4 -> 6.6)
constexpr long long FEW_BYTES = 16ll << 20;
__global__ __launch_bounds__(THREADS) void adam_partial(const AdamTable t, double* __restrict__ part, AdamScalars* __restrict__ held) {
  __shared__ double red[THREADS / 64];
  const int j = entry_of(t.first, t.count, blockIdx.x);
  const long long lo = (long long)((int)blockIdx.x - t.first[j]) * t.chunk;
  const long long left = t.job[j].n - lo;
  const double sum = block_join<RTG_NORM_L2, THREADS>(chunk_sum<float, RTG_NORM_L2, false>(t.job[j].grads + lo, left < t.chunk ? left : t.chunk), red);
  if (threadIdx.x != 0) return;
  part[blockIdx.x] = sum;
  if ((int)blockIdx.x == t.first[j]) held[j] = AdamScalars{t.job[j].step_state[0], 0.f, 0.f, adam_flagged(t.job[j].loss_flag) ? 0.f : 1.f};
}

// FEW: sc is what adam_partial held; else what adam_prepare made.  Parameters, gradients and moments pass the caches by where
// they are many: what the memory-side cache holds is then the gradients that the norm has just read, not the moments of
// buffers that are done with until the next step (27 M parameters 139 us, with plain accesses 26 more).  A small model may fit as
// a whole (2.7 M in the caches 21.1 us, past them 23.6; coming from HBM 26.1 and 23.9).
template <bool FEW>
__global__ __launch_bounds__(THREADS) void adam_update(const AdamTable t, const AdamScalars* __restrict__ sc, const double* __restrict__ part,
                                                       int n_part, const AdamRates rates, float* __restrict__ norm_out, float w1, float b2,
                                                       float w2, float decay, float eps) {
  const int j = entry_of(t.first, t.count, blockIdx.x);
  AdamScalars s = sc[j];
  if constexpr (FEW) {
    __shared__ double red[THREADS / 64];
    const double norm = adam_norm(all_partials<RTG_NORM_L2, THREADS>(part, n_part, red), rates);
    const float before = s.step_size;
    s = adam_scalars(norm, before, s.go == 0.f, rates);
    if (threadIdx.x == 0) {
      if (blockIdx.x == 0 && norm_out) *norm_out = (float)norm;
      if ((int)blockIdx.x == t.first[j] && s.go != 0.f) t.job[j].step_state[0] = before + 1.f;
    }
  }
  if (s.go == 0.f) return;
  const long long lo = (long long)((int)blockIdx.x - t.first[j]) * t.chunk;
  const long long left = t.job[j].n - lo, n = left < t.chunk ? left : t.chunk;
  float* const __restrict__ p = t.job[j].params + lo;
  const float* const __restrict__ g = t.job[j].grads + lo;
  float* const __restrict__ m = t.job[j].exp_avg + lo;
  float* const __restrict__ v = t.job[j].exp_avg_sq + lo;
  const auto step = [&](float& pi, float gi, float& mi, float& vi) __attribute__((always_inline)) {
    gi *= s.scale;
    mi = mi + w1 * (gi - mi);
    vi = vi * b2 + w2 * gi * gi;
    pi = pi * decay - s.step_size * mi / (sqrtf(vi) / s.bc2s + eps);
  };
  const long long nv = n / 4;
  for (long long i = threadIdx.x; i < nv; i += THREADS) {
    RtgVec<float> a, b, c, d;
    rtg_load<!FEW>(a, p + 4 * i);
    rtg_load<!FEW>(b, g + 4 * i);
    rtg_load<!FEW>(c, m + 4 * i);
    rtg_load<!FEW>(d, v + 4 * i);
    float pr[4], mr[4], vr[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pr[e] = a.get(e);
      mr[e] = c.get(e);
      vr[e] = d.get(e);
      step(pr[e], b.get(e), mr[e], vr[e]);
    }
    a.set(pr);
    c.set(mr);
    d.set(vr);
    rtg_store<!FEW>(a, p + 4 * i);
    rtg_store<!FEW>(c, m + 4 * i);
    rtg_store<!FEW>(d, v + 4 * i);
  }
  const long long i = 4 * nv + threadIdx.x;
  if (i < n) step(p[i], g[i], m[i], v[i]);
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
constexpr int MAX_TENSORS = 1 << 20;

constexpr int MOST_GROUPS = 4096;
constexpr long long KB = 1024;
long long up(long long bytes) { return (bytes + 4095) / 4096 * 4096; }

// Bytes of a chunk, and the workgroups that share a launch's chunks (8 a CU, 16 where the list is not in the caches).  Norm /
// clipping of 27 M floats with chunks of 16, 32, 64 KB: 28.4 / 59.7, 25.5 / 57.7, 26.0 / 61.1 us; of 2.7 M 9.7 / 16.0, 9.9 / 16.0,
// 10.4 / 17.4; of 537 M bf16 values in 4096 workgroups 207 / 609, 189 / 585, 185 / 591, in 2048 241 / 655, 214 / 621, 203 / 618.
struct Cut { long long chunk; int groups; };
Cut cut_of(long long total) {
  const long long c = total < 32 * KB * KB ? 16 * KB : total <= CACHED ? 32 * KB : 64 * KB, least = up(total >> 20);
  return {c > least ? c : least, total <= CACHED ? MOST_GROUPS / 2 : MOST_GROUPS};
}

long long list_bytes(int n, const long long* counts, const int* bf16) {
  long long total = 0;
  for (int i = 0; i < n; ++i) total += counts[i] * (bf16[i] ? 2 : 4);
  return total;
}

// walks the list, TABLE tensors a launch: launch(table, workgroups, workgroups before) for each -> status; *blocks: all of them
// (at most MOST_GROUPS a launch)
template <class F>
int each_table(int n, void* const* grads, const long long* counts, const int* bf16, long long total, int* blocks, F launch) {
  const Cut cut = cut_of(total);
  GradTable t;
  t.chunk = cut.chunk;
  int before = 0, here = 0;
  t.count = 0;
  for (int k = 0; k < TABLE / 32; ++k) t.bf16[k] = 0;
  for (int i = 0; i <= n; ++i) {
    if (t.count == TABLE || (i == n && t.count > 0)) {
      t.chunks = here;
      if (here > cut.groups) here = cut.groups;
      const int rc = launch(t, here, before);
      if (rc != RTG_OK) return rc;
      before += here;
      here = t.count = 0;
      for (int k = 0; k < TABLE / 32; ++k) t.bf16[k] = 0;
    }
    if (i == n || counts[i] == 0) continue;
    const long long bytes = counts[i] * (bf16[i] ? 2 : 4);
    t.p[t.count] = grads[i];
    t.n[t.count] = counts[i];
    t.first[t.count] = here;
    if (bf16[i]) t.bf16[t.count >> 5] |= 1u << (t.count & 31);
    here += (int)((bytes + t.chunk - 1) / t.chunk);
    ++t.count;
  }
  *blocks = before;
  return RTG_OK;
}

int check_list(int n, void* const* grads, const long long* counts, const int* bf16, int kind, const void* ws) {
  if (!grads || !counts || !bf16 || !ws) return RTG_ENULL;
  if (n < 1 || n > MAX_TENSORS || (kind != RTG_NORM_L2 && kind != RTG_NORM_MAX)) return RTG_EINVAL;
  long long total = 0;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0) return RTG_EINVAL;
    if (counts[i] > (1ll << 56) || (total += counts[i]) > (1ll << 56)) return RTG_ERANGE;
    if (counts[i] > 0 && !grads[i]) return RTG_ENULL;
    if (reinterpret_cast<uintptr_t>(grads[i]) & (bf16[i] ? 1 : 3)) return RTG_EINVAL;
  }
  return RTG_OK;
}

struct Range { uintptr_t lo, hi; bool written; };
// no two ranges share a byte: workgroups of one launch would write what others read.  A list in the order of its addresses
// (the views of a flat buffer) needs no sorting.
int disjoint(Range* r, long long n) {
  const auto ordered = [&]() {
    for (long long i = 1; i < n; ++i)
      if (r[i - 1].hi > r[i].lo) return false;
    return true;
  };
  if (ordered()) return RTG_OK;
  std::sort(r, r + n, [](const Range& a, const Range& b) { return a.lo < b.lo; });
  return ordered() ? RTG_OK : RTG_EINVAL;
}

// the float at p shares a byte with a range that is written (r: disjoint, so in the order of the addresses)
bool is_written(const Range* r, long long n, const float* p) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  for (const Range* q = std::upper_bound(r, r + n, lo + 3, [](uintptr_t at, const Range& a) { return at < a.lo; }); q > r;) {
    --q;
    if (q->hi > lo) {
      if (q->written) return true;
    } else if (q->hi > q->lo) {
      break;                                               // (empty ranges are passed over)
    }
  }
  return false;
}

template <int KIND>
int partials(int n, void* const* grads, const long long* counts, const int* bf16, long long total, double* ws, int* blocks, hipStream_t st) {
  return each_table(n, grads, counts, bf16, total, blocks, [&](const GradTable& t, int here, int before) {
    if (total > CACHED) RTG_KLAUNCH((grad_partial<KIND, true>), dim3(here), dim3(THREADS), 0, st, t, ws + before);
    else RTG_KLAUNCH((grad_partial<KIND, false>), dim3(here), dim3(THREADS), 0, st, t, ws + before);
    return rtg_launch_status();
  });
}

template <int KIND>
int norm(int n, void* const* grads, const long long* counts, const int* bf16, double* ws, float* out, hipStream_t st) {
  int blocks = 0;
  const int rc = partials<KIND>(n, grads, counts, bf16, list_bytes(n, counts, bf16), ws, &blocks, st);
  if (rc != RTG_OK) return rc;
  RTG_KLAUNCH(grad_norm_finish<KIND>, dim3(1), dim3(REDUCE), 0, st, ws, blocks, out, 0);
  return rtg_launch_status();
}

template <int KIND>
int clip(int n, void* const* grads, const long long* counts, const int* bf16, double max_norm, double* ws, float* out, hipStream_t st) {
  const long long total = list_bytes(n, counts, bf16);
  int blocks = 0, again = 0;
  const int rc = partials<KIND>(n, grads, counts, bf16, total, ws, &blocks, st);
  if (rc != RTG_OK) return rc;
  const bool first = blocks == 0 || blocks > JOIN_FIRST;      // (nothing but empty tensors: the norm is 0)
  if (first) {
    RTG_KLAUNCH(grad_norm_finish<KIND>, dim3(1), dim3(REDUCE), 0, st, ws, blocks, out, (int)(blocks > 0));
    const int joined = rtg_launch_status();
    if (joined != RTG_OK || blocks == 0) return joined;
  }
  return each_table(n, grads, counts, bf16, total, &again, [&](const GradTable& t, int here, int before) {
    const int parts = first ? 1 : blocks, write_norm = before == 0 && !first;
    if (total > CACHED)
      RTG_KLAUNCH((grad_scale<KIND, false>), dim3(here), dim3(THREADS), 0, st, t, (const double*)ws, parts, max_norm, out, write_norm);
    else
      RTG_KLAUNCH((grad_scale<KIND, true>), dim3(here), dim3(THREADS), 0, st, t, (const double*)ws, parts, max_norm, out, write_norm);
    return rtg_launch_status();
  });
}

long long most_partials(int n) { return (long long)MOST_GROUPS * ((n + TABLE - 1) / TABLE); }

}  // namespace

extern "C" long long rtg_grad_ws(int n) {
  if (n < 1 || n > MAX_TENSORS) return RTG_EINVAL;
  // a partial per workgroup, and AdamW's scalars
  return most_partials(n) + (long long)n * (sizeof(AdamScalars) / sizeof(double));
}

extern "C" int rtg_grad_norm(int n, const void* const* grads, const long long* counts, const int* bf16, int kind, double* ws,
                             float* norm_out, void* stream) {
  void* const* g = const_cast<void* const*>(grads);
  const int rc = check_list(n, g, counts, bf16, kind, ws);
  if (rc != RTG_OK) return rc;
  if (!norm_out) return RTG_ENULL;
  return kind == RTG_NORM_L2 ? norm<RTG_NORM_L2>(n, g, counts, bf16, ws, norm_out, (hipStream_t)stream)
                             : norm<RTG_NORM_MAX>(n, g, counts, bf16, ws, norm_out, (hipStream_t)stream);
}

extern "C" int rtg_grad_clip(int n, void* const* grads, const long long* counts, const int* bf16, int kind, double max_norm, double* ws,
                             float* norm_out, void* stream) {
  const int rc = check_list(n, grads, counts, bf16, kind, ws);
  if (rc != RTG_OK) return rc;
  if (!norm_out) return RTG_ENULL;
  if (!(max_norm >= 0.0)) return RTG_EINVAL;
  {
    std::unique_ptr<Range[]> r(new (std::nothrow) Range[n]);
    if (!r) return RTG_ERANGE;
    int k = 0;
    for (int i = 0; i < n; ++i) {
      const uintptr_t lo = reinterpret_cast<uintptr_t>(grads[i]);
      if (counts[i] > 0) r[k++] = Range{lo, lo + (uintptr_t)counts[i] * (bf16[i] ? 2 : 4), true};
    }
    const int apart = disjoint(r.get(), k);
    if (apart != RTG_OK) return apart;
    if (is_written(r.get(), k, norm_out)) return RTG_EINVAL;
  }
  return kind == RTG_NORM_L2 ? clip<RTG_NORM_L2>(n, grads, counts, bf16, max_norm, ws, norm_out, (hipStream_t)stream)
                             : clip<RTG_NORM_MAX>(n, grads, counts, bf16, max_norm, ws, norm_out, (hipStream_t)stream);
}

extern "C" int rtg_adamw_clipped(int n, const RtgAdamWJob* jobs, double max_norm, double lr, double beta1, double beta2, double eps,
                                 double weight_decay, float grad_scale, double* ws, float* norm_out, void* stream) {
  if (!jobs || !ws) return RTG_ENULL;
  if (n < 1 || n > MAX_TENSORS || !(max_norm >= 0.0)) return RTG_EINVAL;
  long long total = 0;
  for (int i = 0; i < n; ++i) {
    const RtgAdamWJob& j = jobs[i];
    if (!j.params || !j.grads || !j.exp_avg || !j.exp_avg_sq || !j.step_state) return RTG_ENULL;
    if (j.n < 1) return RTG_EINVAL;
    if (j.n > (1ll << 56) || (total += j.n) > (1ll << 56)) return RTG_ERANGE;
    if ((reinterpret_cast<uintptr_t>(j.params) | reinterpret_cast<uintptr_t>(j.grads) | reinterpret_cast<uintptr_t>(j.exp_avg) |
         reinterpret_cast<uintptr_t>(j.exp_avg_sq) | reinterpret_cast<uintptr_t>(j.step_state)) & 3) return RTG_EINVAL;
  }
  {
    std::unique_ptr<Range[]> r(new (std::nothrow) Range[5 * (size_t)n + 1]);
    if (!r) return RTG_ERANGE;
    for (int i = 0; i < n; ++i) {
      const RtgAdamWJob& j = jobs[i];
      const void* p[5] = {j.params, j.exp_avg, j.exp_avg_sq, j.step_state, j.grads};
      for (int k = 0; k < 5; ++k) {
        const uintptr_t lo = reinterpret_cast<uintptr_t>(p[k]);
        r[5 * (size_t)i + k] = Range{lo, lo + (k != 3 ? 4 * (uintptr_t)j.n : 4), k < 4};
      }
    }
    const uintptr_t out = reinterpret_cast<uintptr_t>(norm_out);
    r[5 * (size_t)n] = Range{out, out + (out ? 4 : 0), true};
    const int apart = disjoint(r.get(), 5ll * n + 1);
    if (apart != RTG_OK) return apart;
    // (the flags of later buffers are read when earlier ones have been updated)
    const float* last = nullptr;
    for (int i = 0; i < n; ++i) {
      const float* flag = jobs[i].loss_flag;
      if (flag && flag != last && is_written(r.get(), 5ll * n + 1, flag)) return RTG_EINVAL;
      last = flag;
    }
  }
  hipStream_t st = (hipStream_t)stream;
  const AdamRates rates{max_norm, lr, beta1, beta2, grad_scale};
  const float w1 = (float)(1.0 - beta1), w2 = (float)(1.0 - beta2), decay = (float)(1.0 - lr * weight_decay);
  AdamScalars* sc = reinterpret_cast<AdamScalars*>(ws + most_partials(n));
  const Cut cut = cut_of(4 * total);
  // The update in smaller pieces than the norm: four streams in, three out, and no partial a piece.  A vector of each a thread
  // (27 M parameters 143 us, in pieces of 16 KB 147; 84 M 413 and 431, in 8192 pieces 454); where every workgroup joins the
  // partials first, four, but a workgroup for each CU where there is that much (2.7 M 21.1 us, in pieces of 4 KB 24.7; 0.2 M
  // 9.7 and 8.2).
  const long long least = up(total >> 18), few = up(total >> 6);
  AdamTable a;
  const auto fill = [&](int from, long long bytes) {           // -> workgroups
    int here = 0;
    a.chunk = bytes / 4;
    for (a.count = 0; a.count < JOBS && from + a.count < n; ++a.count) {
      a.job[a.count] = jobs[from + a.count];
      a.first[a.count] = here;
      here += (int)((jobs[from + a.count].n + a.chunk - 1) / a.chunk);
    }
    return here;
  };
  if (n <= JOBS && 4 * total <= FEW_BYTES) {
    const int blocks = fill(0, cut.chunk);
    RTG_KLAUNCH(adam_partial, dim3(blocks), dim3(THREADS), 0, st, a, ws, sc);
    const int rc = rtg_launch_status();
    if (rc != RTG_OK) return rc;
    const int here = fill(0, few < 4096 ? 4096 : few > 16384 ? 16384 : few);
    RTG_KLAUNCH(adam_update<true>, dim3(here), dim3(THREADS), 0, st, a, (const AdamScalars*)sc, (const double*)ws, blocks, rates, norm_out,
                w1, (float)beta2, w2, decay, (float)eps);
    return rtg_launch_status();
  }
  // the partials, TABLE buffers a launch (in the caches whatever their size: the update reads past them, and a part stays: 84 M
  // parameters 491 -> 454 us)
  GradTable t;
  t.chunk = cut.chunk;
  for (int k = 0; k < TABLE / 32; ++k) t.bf16[k] = 0;
  int blocks = 0;
  for (int i = 0; i < n; i += TABLE) {
    int here = 0;
    for (t.count = 0; t.count < TABLE && i + t.count < n; ++t.count) {
      const RtgAdamWJob& j = jobs[i + t.count];
      t.p[t.count] = const_cast<float*>(j.grads);
      t.n[t.count] = j.n;
      t.first[t.count] = here;
      here += (int)((4 * j.n + t.chunk - 1) / t.chunk);
    }
    t.chunks = here;
    if (here > cut.groups) here = cut.groups;
    RTG_KLAUNCH((grad_partial<RTG_NORM_L2, false>), dim3(here), dim3(THREADS), 0, st, t, ws + blocks);
    const int rc = rtg_launch_status();
    if (rc != RTG_OK) return rc;
    blocks += here;
  }
  for (int i = 0; i < n; i += JOBS) {
    const int here = fill(i, least < 4096 ? 4096 : least);
    RTG_KLAUNCH(adam_prepare, dim3(1), dim3(REDUCE), 0, st, a, (const double*)ws, blocks, rates, sc + i, norm_out, (int)(i == 0));
    int rc = rtg_launch_status();
    if (rc != RTG_OK) return rc;
    RTG_KLAUNCH(adam_update<false>, dim3(here), dim3(THREADS), 0, st, a, (const AdamScalars*)(sc + i), (const double*)nullptr, 0, rates,
                (float*)nullptr, w1, (float)beta2, w2, decay, (float)eps);
    rc = rtg_launch_status();
    if (rc != RTG_OK) return rc;
  }
  return RTG_OK;
}

// Softmax of scores with a learned relative-position bias, and its gradient.
//
//   l = scale s + table[bucket(k - pos), head],  pos = query + offset[batch]
//   over the keys k < length[batch] (and k <= pos when causal);
//   p = D(exp(l - lse)),  lse = log sum exp l,  D dropout; a row without keys
//   gives zeros and lse = -inf.
//   Gradient: P = exp(l - lse), d = D(dp), dl = P (d - sum P d), ds = scale dl,
//   dtable[b, head] = sum of dl where the bucket is b.
//
// bucket(rel): the number of thresholds that are at most the distance |rel|
// (bidirectional; the buckets of rel > 0 follow those of rel <= 0) or
// max(-rel, 0).  From the last threshold W on the bucket stays the same, so a
// row meets a window of less than 2W distances and two constants outside it.
// A CTA works on one head: it looks the table up once, into a shared array of
// the window by distance.  In the gradient a row holds each distance of the
// window once, so its owner adds dl to the window's sum without atomics, in row
// order; what lies outside is summed in registers.  Buckets are ranges of
// the window: they are folded once at the end, into a partial sum for each
// CTA that a second kernel adds in CTA order.
//
// Rows start anywhere (any number of keys): a row is read and written in the
// tensor's own aligned 16-byte units, whose first and last may hold elements of
// the neighbouring rows; those are masked, and only such cut units are stored
// element by element.  Units without a visible key are not read.
//
// exp(l - m) is 2^(l L - RN(m L)) with L = log2 e: an element costs a fused
// multiply-add for its logit, one for the exponent and ex2.approx (relative
// error 2^-22).  The rounding of m L is one factor for all that share m.
// Where m L could overflow (|m| > 2^100: rows at the type's lowest value) the
// difference is taken first.  Each warp takes its own maximum, and its sum is
// rescaled when the team's records meet: one exchange a row.
#include <cuda_runtime.h>

#include <algorithm>

#include "act_io.cuh"
#include "kernels.h"
#include "pdl.cuh"
#include "philox.cuh"
#include "row_team.cuh"

namespace askb {

namespace {

constexpr int kWarpTeamThreads = 256;
constexpr float kNegInf = -__builtin_huge_valf();

// The window's geometry: distances rel in [-W, hi] at index rel + W.
struct Window {
  int w, hi, size;
};
__host__ __device__ inline Window window_of(const BiasSoftmaxArgs& a) {
  const int w = a.n_thresholds ? a.thresholds[a.n_thresholds - 1] : 0;
  const int hi = a.bidirectional ? w : 0;
  return Window{w, hi, w + hi + 1};
}

__device__ __forceinline__ int bucket_of(const BiasSoftmaxArgs& a, int rel) {
  const int n = a.bidirectional ? abs(rel) : max(-rel, 0);
  int lo = 0, hi = a.n_thresholds;  // thresholds[0, lo) <= n < thresholds[hi, ..)
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.thresholds[mid] <= n) lo = mid + 1; else hi = mid;
  }
  return a.bidirectional && rel > 0 ? lo + a.n_thresholds + 1 : lo;
}

// The head's bias by distance.
__device__ __forceinline__ void fill_window(const BiasSoftmaxArgs& a, const Window& win, uint32_t head, float* lut) {
  for (int i = int(threadIdx.x); i < win.size; i += int(blockDim.x)) {
    float v[1];
    param_load<1>(a.table, a.table_type, uint64_t(bucket_of(a, i - win.w)) * a.heads + head, v);
    lut[i] = v[0];
  }
}

// One row as the team sees it.
struct Row {
  uint64_t index;      // of the row
  uint64_t first;      // element index of its first unit
  int shift;           // elements of that unit before the row
  int pos, visible;    // query position; keys [0, visible) are seen
};
template <int V>
__device__ __forceinline__ Row row_of(const BiasSoftmaxArgs& a, uint32_t head, uint64_t pair) {
  Row r;
  const uint64_t b = pair / a.queries, q = pair - b * a.queries;
  r.index = (b * a.heads + head) * a.queries + q;
  const uint64_t e = r.index * a.keys;
  r.shift = int(e % uint64_t(V));
  r.first = e - uint64_t(r.shift);
  const int64_t pos = int64_t(q) + (a.offsets ? int64_t(__ldg(a.offsets + b)) : 0);
  int64_t seen = a.keys;
  if (a.lengths) seen = min(seen, int64_t(__ldg(a.lengths + b)));
  if (a.causal) seen = min(seen, pos + 1);
  r.visible = int(max(seen, int64_t(0)));
  // far positions meet only the window's ends, whatever their distance
  r.pos = int(max(min(pos, int64_t(1) << 30), -(int64_t(1) << 30)));
  return r;
}

// The unit's elements of `p`, where any is visible.
template <int T, int V>
__device__ __forceinline__ void load_seen(const BiasSoftmaxArgs& a, const void* p, const Row& r, int k0, uint64_t total,
                                          float* v) {
  const uint64_t at = r.first + uint64_t(int64_t(k0) + r.shift);
  if (k0 >= r.visible || k0 + V <= 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.0f;
  } else if (a.aligned && at + V <= total) {
    ActRaw<T, V> raw;
    raw.load(p, at);
    raw.widen(v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = k0 + j >= 0 && k0 + j < r.visible ? act_load<T>(p, at + j) : 0.0f;
  }
}
// The unit's elements that belong to the row.
template <int T, int V>
__device__ __forceinline__ void store_row(const BiasSoftmaxArgs& a, const Row& r, int k0, const float* v) {
  if (k0 >= int(a.keys)) return;
  const uint64_t at = r.first + uint64_t(int64_t(k0) + r.shift);
  if (a.aligned && k0 >= 0 && k0 + V <= int(a.keys)) {
    act_put<T, V>(a.out, at, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (k0 + j >= 0 && k0 + j < int(a.keys)) act_store<T>(a.out, at + j, v[j]);
  }
}

// x[j] <- scale x[j] + bias where the key is visible, else -inf.
template <int V>
__device__ __forceinline__ void biased(const Row& r, const Window& win, const float* lut, float scale, int k0, float* x) {
  const int rel = k0 - r.pos;
  if (k0 >= r.visible || k0 + V <= 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = kNegInf;
    return;
  }
  if (rel >= win.hi || rel + V - 1 <= -win.w) {
    const float b = lut[rel >= win.hi ? win.size - 1 : 0];
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = __fmaf_rn(x[j], scale, b);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = __fmaf_rn(x[j], scale, lut[min(max(rel + j, -win.w), win.hi) + win.w]);
  }
  if (k0 < 0 || k0 + V > r.visible) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (k0 + j < 0 || k0 + j >= r.visible) x[j] = kNegInf;
  }
}

// v <- exp(v - m); v may be -inf, m is not.
template <int E>
__device__ __forceinline__ void exp_minus(float (&v)[E], float m) {
  if (fabsf(m) <= 0x1p100f) {
    const float nm = -m * kLog2e;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = ex2_approx(__fmaf_rn(v[i], kLog2e, nm));
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = ex2_approx((v[i] - m) * kLog2e);
  }
}

struct Task {
  uint32_t head;
  uint64_t pair, end, step;
};
__device__ __forceinline__ Task task_of(const BiasSoftmaxArgs& a, const Team& t) {
  const bool warp_teams = a.shape.warp_teams;
  const uint32_t place = blockIdx.x / t.ctas, chunk = place / a.heads;
  const uint64_t n = a.batch * a.queries;
  Task k;
  k.head = place % a.heads;
  k.pair = n * chunk / a.chunks + (warp_teams ? threadIdx.x >> 5 : 0);
  k.end = n * (chunk + 1) / a.chunks;
  k.step = warp_teams ? blockDim.x >> 5 : 1;
  return k;
}

template <int T, int VPT>
__global__ void __launch_bounds__(kTeamThreads) bias_softmax_kernel(const __grid_constant__ BiasSoftmaxArgs a) {
  constexpr int V = act_vec<T>(), E = V * VPT;
  extern __shared__ float lut[];
  __shared__ TeamRecords<2> sh;
  const Team t = team_of(a.shape.warp_teams);
  const Window win = window_of(a);
  Task task = task_of(a, t);
  pdl_enter();
  team_start(t);
  fill_window(a, win, task.head, lut);
  __syncthreads();
  const DropRun run = drop_run(a.drop, a.seed);
  const uint64_t total = a.batch * a.heads * a.queries * a.keys;
  for (int parity = 0; task.pair < task.end; task.pair += task.step, parity ^= 1) {
    const Row r = row_of<V>(a, task.head, task.pair);
    auto key = [&](int q) { return int(((t.rank * VPT + q) * t.threads + t.tid) * uint32_t(V)) - r.shift; };
    float e[E];
#pragma unroll
    for (int q = 0; q < VPT; ++q) load_seen<T, V>(a, a.s, r, key(q), total, e + q * V);
    float m = kNegInf;
#pragma unroll
    for (int q = 0; q < VPT; ++q) {
      biased<V>(r, win, lut, a.scale, key(q), e + q * V);
#pragma unroll
      for (int j = 0; j < V; ++j) m = fmaxf(m, e[q * V + j]);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float base = m == kNegInf ? 0.0f : m;  // nothing visible: every 2^x below is 0
    float s = 0.0f;
    exp_minus<E>(e, base);
#pragma unroll
    for (int i = 0; i < E; ++i) s += e[i];
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    // the team's maximum and sum from the warps' own
    float top = base, sum = s, factor = 1.0f;
    const uint32_t records = t.warps * t.ctas;
    if (records > 1) {
      const float rec[2] = {m, s};
      team_exchange<2>(t, sh, parity, rec);
      top = kNegInf;
      for (uint32_t k = 0; k < records; ++k) top = fmaxf(top, sh.v[parity][k][0]);
      if (top == kNegInf) top = 0.0f;
      sum = 0.0f;
      for (uint32_t k = 0; k < records; ++k) sum = __fmaf_rn(sh.v[parity][k][1], ex2_approx((sh.v[parity][k][0] - top) * kLog2e), sum);
      factor = ex2_approx((m - top) * kLog2e);
    }
    factor = sum == 0.0f ? 0.0f : factor * __frcp_rn(sum);
    if (t.tid == 0 && t.rank == 0) a.lse[r.index] = sum == 0.0f ? kNegInf : top + logf(sum);
#pragma unroll
    for (int q = 0; q < VPT; ++q) {
      const int k0 = key(q);
      float* v = e + q * V;
      const bool seen = k0 < r.visible && k0 + V > 0;
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = k0 + j >= 0 && k0 + j < r.visible ? v[j] * factor : 0.0f;
      if (a.drop.on && seen) drop_unit<V>(run, r.first + uint64_t(int64_t(k0) + r.shift), v);
      store_row<T, V>(a, r, k0, v);
    }
  }
}

template <int T, int VPT>
__global__ void __launch_bounds__(kTeamThreads) bias_softmax_grad_kernel(const __grid_constant__ BiasSoftmaxArgs a) {
  constexpr int V = act_vec<T>(), E = V * VPT;
  extern __shared__ float lut[];
  __shared__ TeamRecords<1> sh;
  __shared__ float ends[2][kTeamThreads / 32];
  const bool warp_teams = a.shape.warp_teams;
  const Team t = team_of(a.shape.warp_teams);
  const Window win = window_of(a);
  Task task = task_of(a, t);
  const int teams = warp_teams ? int(blockDim.x >> 5) : 1;
  float* const sums = lut + win.size;  // the teams' windows
  float* const mine = sums + (warp_teams ? int(threadIdx.x >> 5) : 0) * win.size;
  pdl_enter();
  team_start(t);
  fill_window(a, win, task.head, lut);
  for (int i = int(threadIdx.x); i < teams * win.size; i += int(blockDim.x)) sums[i] = 0.0f;
  __syncthreads();
  const DropRun run = drop_run(a.drop, a.seed);
  const uint64_t total = a.batch * a.heads * a.queries * a.keys;
  float left = 0.0f, right = 0.0f;  // dl at rel <= -W and at rel >= hi
  for (int parity = 0; task.pair < task.end; task.pair += task.step, parity ^= 1) {
    const Row r = row_of<V>(a, task.head, task.pair);
    auto key = [&](int q) { return int(((t.rank * VPT + q) * t.threads + t.tid) * uint32_t(V)) - r.shift; };
    float p[E], d[E];
#pragma unroll
    for (int q = 0; q < VPT; ++q) {
      load_seen<T, V>(a, a.s, r, key(q), total, p + q * V);
      load_seen<T, V>(a, a.dp, r, key(q), total, d + q * V);
    }
    const float lse = __ldg(a.lse_in + r.index);
    const float base = lse == kNegInf ? 0.0f : lse;  // all logits are -inf then, and every P is 0
    float dot[1] = {0.0f};
#pragma unroll
    for (int q = 0; q < VPT; ++q) {
      const int k0 = key(q);
      biased<V>(r, win, lut, a.scale, k0, p + q * V);
      if (a.drop.on && k0 < r.visible && k0 + V > 0)
        drop_unit<V>(run, r.first + uint64_t(int64_t(k0) + r.shift), d + q * V);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = q * V + j;
        const bool seen = k0 + j >= 0 && k0 + j < r.visible;
        d[i] = seen ? d[i] : 0.0f;
      }
    }
    exp_minus<E>(p, base);
#pragma unroll
    for (int i = 0; i < E; ++i) dot[0] = __fmaf_rn(p[i], d[i], dot[0]);
    team_sum<1>(t, sh, parity, dot);
    if (warp_teams) __syncwarp();  // the lanes' adds of the row before are done
    float row_left = 0.0f, row_right = 0.0f;
#pragma unroll
    for (int q = 0; q < VPT; ++q) {
      const int k0 = key(q), rel = k0 - r.pos;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = q * V + j;
        const bool seen = k0 + j >= 0 && k0 + j < r.visible;
        p[i] = seen ? p[i] * (d[i] - dot[0]) : 0.0f;
        o[j] = p[i] * a.scale;
        if (seen) {
          if (rel + j <= -win.w) row_left += p[i];
          else if (rel + j >= win.hi) row_right += p[i];
          else mine[rel + j + win.w] += p[i];
        }
      }
      store_row<T, V>(a, r, k0, o);
    }
    left += row_left;
    right += row_right;
  }
  // fold the windows by bucket
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    left += __shfl_xor_sync(0xffffffffu, left, d);
    right += __shfl_xor_sync(0xffffffffu, right, d);
  }
  const int warp = int(threadIdx.x >> 5), lane = int(threadIdx.x & 31u), warps = int(blockDim.x >> 5);
  if (lane == 0) {
    ends[0][warp] = left;
    ends[1][warp] = right;
  }
  __syncthreads();
  const int side = a.n_thresholds + 1;
  for (int b = warp; b < int(a.buckets); b += warps) {
    const bool ahead = b >= side;  // rel > 0
    const int j = ahead ? b - side : b;
    // distances [n0, n1) of the bucket, inside the window
    const int n0 = max(j ? a.thresholds[j - 1] : 0, ahead ? 1 : 0), n1 = j < a.n_thresholds ? a.thresholds[j] : win.w;
    float v = 0.0f;
    for (int k = 0; k < teams; ++k)
      for (int n = n0 + lane; n < n1; n += 32) {
        const int at = ahead ? win.w + n : win.w - n;
        if (at > 0 && at < win.size - 1) v += sums[k * win.size + at];
      }
    const bool is_left = !ahead && j == a.n_thresholds, is_right = a.bidirectional ? ahead && j == a.n_thresholds : j == 0;
    if (lane < warps) v += (is_left ? ends[0][lane] : 0.0f) + (is_right ? ends[1][lane] : 0.0f);
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (lane == 0) a.partial[uint64_t(blockIdx.x) * a.buckets + b] = v;
  }
}

// dtable[b, head]: a warp adds the head's CTAs in order of their chunks.
__global__ void __launch_bounds__(256) bias_table_join_kernel(const float* __restrict__ partial, float* __restrict__ dtable,
                                                              uint32_t heads, uint32_t buckets, uint32_t chunks,
                                                              uint32_t ctas) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t out = uint64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (out >= uint64_t(heads) * buckets) return;
  const uint32_t b = uint32_t(out / heads), head = uint32_t(out % heads);
  double v = 0.0;
  for (uint32_t k = lane; k < chunks * ctas; k += 32) {
    const uint64_t cta = (uint64_t(k / ctas) * heads + head) * ctas + k % ctas;
    v += double(partial[cta * buckets + b]);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (lane == 0) dtable[out] = float(v);
}

template <int T>
const void* kernel_of_type(int elems, bool grad) {
  constexpr int V = act_vec<T>();
  if (grad)
    return elems == 8    ? (const void*)bias_softmax_grad_kernel<T, 8 / V>
           : elems == 16 ? (const void*)bias_softmax_grad_kernel<T, 16 / V>
                         : (const void*)bias_softmax_grad_kernel<T, 32 / V>;
  return elems == 8    ? (const void*)bias_softmax_kernel<T, 8 / V>
         : elems == 16 ? (const void*)bias_softmax_kernel<T, 16 / V>
                       : (const void*)bias_softmax_kernel<T, 32 / V>;
}
const void* kernel_for(const BiasSoftmaxArgs& a, bool grad) {
  return a.type == kF32 ? kernel_of_type<kF32>(a.shape.elems, grad)
         : a.type == kF16 ? kernel_of_type<kF16>(a.shape.elems, grad) : kernel_of_type<kBF16>(a.shape.elems, grad);
}

// Windows above the default 48 KB (static arrays included) need the kernel's limit raised.
cudaError_t allow_shared(const void* kernel, uint32_t bytes) {
  return bytes <= 32 * 1024 ? cudaSuccess
                            : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
}

constexpr uint32_t kWindowBytes = 192 * 1024;  // dynamic shared memory of a CTA at most

}  // namespace

TeamShape bias_softmax_shape(uint64_t keys, uint64_t rows, int type, bool grad, int sms) {
  (void)grad;
  const uint64_t v = type == kF32 ? 4 : 8;
  // a row that starts inside a unit spreads over one more
  const uint64_t span = keys % v ? keys + v - 1 : keys;
  TeamShape s{0, kWarpTeamThreads, 1, 32};
  if (rows >= uint64_t(sms) * 8 && span <= 32 * 32) {
    s.warp_teams = 32;
    s.elems = span <= 32 * 8 ? 8 : span <= 32 * 16 ? 16 : 32;
    return s;
  }
  if (rows < uint64_t(sms) * 2) s.elems = 8;  // few rows: more threads for each
  while (s.elems < 32 && span > uint64_t(kTeamThreads) * s.elems) s.elems *= 2;
  // few rows: spread each over a cluster while SMs idle and every CTA keeps 256 threads' worth of a row
  while (s.ctas < kTeamCluster &&
         (span > uint64_t(kTeamThreads) * s.elems * s.ctas ||
          (rows * s.ctas * 2 <= uint64_t(sms) && span >= uint64_t(512) * s.elems * s.ctas)))
    s.ctas *= 2;
  const uint64_t per = uint64_t(s.elems) * s.ctas;
  s.threads = int(std::max<uint64_t>(32, ((span + per - 1) / per + 31) / 32 * 32));
  return s;
}

void bias_softmax_shared(BiasSoftmaxArgs* a, bool grad) {
  const uint32_t window = uint32_t(window_of(*a).size) * 4;
  uint32_t teams = a->shape.warp_teams ? uint32_t(a->shape.threads) / 32 : 1;
  if (grad && a->shape.warp_teams) {
    while (teams > 1 && window * (1 + teams) > kWindowBytes) --teams;
    a->shape.threads = int(teams) * 32;
  }
  a->shared_bytes = window * (grad ? 1 + teams : 1);
}

cudaError_t bias_softmax_occupancy(const BiasSoftmaxArgs& a, bool grad, int* blocks_per_sm) {
  const void* kernel = kernel_for(a, grad);
  const cudaError_t e = allow_shared(kernel, a.shared_bytes);
  if (e != cudaSuccess) return e;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(blocks_per_sm, kernel, a.shape.threads, a.shared_bytes);
}

cudaError_t bias_softmax_launch(const BiasSoftmaxArgs& a, bool grad, cudaStream_t stream) {
  const uint64_t pairs = a.batch * a.queries;
  if (pairs && a.heads) {
    const void* kernel = kernel_for(a, grad);
    cudaError_t e = allow_shared(kernel, a.shared_bytes);
    if (e != cudaSuccess) return e;
    BiasSoftmaxArgs args = a;
    void* params[] = {&args};
    e = launch_rows(kernel, a.shape, a.heads * a.chunks * unsigned(a.shape.ctas), a.shared_bytes, params, stream);
    if (e != cudaSuccess) return e;
  }
  const uint64_t entries = uint64_t(a.heads) * a.buckets;
  if (!grad || !entries) return cudaSuccess;
  (void)launch_pdl(&bias_table_join_kernel, dim3(unsigned((entries + 7) / 8)), dim3(256), stream,
                   static_cast<const float*>(a.partial), a.dtable, a.heads, a.buckets, pairs ? a.chunks : 0u,
                   uint32_t(a.shape.ctas));
  return cudaGetLastError();
}

}  // namespace askb

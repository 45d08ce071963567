// sy_sample.cu -- one token a row from logits and given random numbers.
//
// Weights are whole numbers, exp(x - max) in units of 2^-40, so every sum is
// exact whatever its order: blocks add in parallel, with atomics, and the token
// does not depend on how they were scheduled.
//
// A cluster of up to 8 CTAs has a row; each keeps its slice of the scaled logits
// in shared memory, so DRAM is read once (slices that do not fit are read again
// from global memory). Tokens are ranked by (x, then lowest index), written as
// one 64-bit number, their rank key; "the first k" and "the first with weight
// p Z" are then "every rank key from some cut on". To find a cut, all tokens are
// counted and weighed in 2048 bins of equal width in max - x (weights beyond
// 28.4 are zero); the bin that holds the cut has a few tokens, as a rule, which
// are gathered and ranked by comparing all pairs. A bin with more than kList of
// them (ties, flat rows) is cut by eight radix passes over the rank keys instead.
// The draw then adds the kept weights in index order: CTAs, warps, lanes.
//
// The row's bytes are the floor for many rows (256 x 131071 fp32: 20.5 us at the
// measured copy rate); for one row it is a chain of about ten cluster barriers.
#include <cooperative_groups.h>

#include <cmath>

#include "sy_common.cuh"
#include "sy_launch.cuh"
#include "sy_serving.cuh"

namespace cg = cooperative_groups;

namespace sy {
namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048, kList = 1024;
constexpr int kMaxCluster = 8;
constexpr float kSpan = 28.43f;                      // exp(-kSpan) 2^40 rounds to 0
constexpr float kBinsPer = (kBins - 1) / kSpan;      // bins per unit of max - x
constexpr int64_t kMaxSlice = 128 * 1024;            // bytes of a slice in shared memory

struct State {
  u64 wbin[kBins];       // weight per bin
  unsigned cbin[kBins];  // tokens per bin
  u64 list[kList], sorted[kList];
  unsigned listed;
  float max_x;
  unsigned max_at;
  u64 total;             // this CTA's kept weight
  // what the leader found, read by the others
  int bin;
  unsigned need;         // tokens (or 0: weight) of the bin up to the cut
  u64 goal, cut;
  u64 red[kWarps];
  float fred[kWarps];
  unsigned ured[kWarps];
};

// x as an order-preserving 32-bit number; the rank key adds the index, lowest first
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);  // -0 ranks with +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 rank_key(float x, unsigned i) {
  return (u64)key_of(x) << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float x_of(u64 rank) {
  const unsigned k = (unsigned)(rank >> 32);
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// exp(x - top), 1 where x is the maximum (infinities included)
__device__ __forceinline__ float mass_of(float x, float top) {
  return x == top ? 1.f : expf(__fsub_rn(x, top));
}
__device__ __forceinline__ u64 weight_of(float e) {
  return __float2ull_rn(__fmul_rn(e, 1099511627776.f));  // 2^40
}
// the bin of x, or kBins where the weight is zero
__device__ __forceinline__ int bin_of(float x, float top) {
  const float d = x == top ? 0.f : __fsub_rn(top, x);
  return d <= kSpan ? (int)(d * kBinsPer) : kBins;
}

__device__ __forceinline__ u64 warp_sum64(u64 x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
  return x;
}
__device__ __forceinline__ u64 block_sum64(u64 x, u64* red) {
  x = warp_sum64(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  u64 s = 0;
#pragma unroll 4
  for (int w = 0; w < kWarps; ++w) s += red[w];
  return s;
}
// exclusive prefix over the block
__device__ __forceinline__ u64 block_before64(u64 x, u64* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 z = __shfl_up_sync(kFull, y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 31) red[warp] = y;
  __syncthreads();
  u64 before = y - x;
#pragma unroll 4
  for (int w = 0; w < kWarps; ++w)
    if (w < warp) before += red[w];
  return before;
}

template <typename T>
struct Slice {
  const T* row;
  float* x;      // shared memory, or nullptr
  unsigned first, count;
  float inv_t;
  __device__ __forceinline__ float scaled(T v) const {
    const float y = __fmul_rn(Dt<T>::to_f(v), inv_t);
    return y == y ? y : -INFINITY;
  }
  __device__ __forceinline__ float at(unsigned i) const { return x ? x[i] : scaled(row[first + i]); }
};

// Read the slice: the maximum and its lowest place; x goes to shared memory.
template <typename T>
__device__ __forceinline__ void read_slice(const Slice<T>& s, float& top, unsigned& at) {
  constexpr int VEC = 16 / (int)sizeof(T);
  top = -INFINITY;
  at = 0xffffffffu;
  auto see = [&](unsigned i, T v) {
    const float y = s.scaled(v);
    if (s.x) s.x[i] = y;
    if (y > top || (y == top && i < at)) top = y, at = i;
  };
  const T* p = s.row + s.first;
  // to the first 16-byte boundary, then whole chunks, four in flight, then the rest
  const unsigned head =
      min(s.count, (unsigned)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (unsigned)sizeof(T));
  if (threadIdx.x < head) see(threadIdx.x, p[threadIdx.x]);
  const unsigned chunks = (s.count - head) / VEC;
  const uint4* q = reinterpret_cast<const uint4*>(p + head);
#pragma unroll 1
  for (unsigned c = threadIdx.x; c < chunks; c += 4 * kThreads) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c + u * kThreads < chunks) v[u] = __ldcs(q + c + u * kThreads);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c + u * kThreads < chunks) {
        const T* e = reinterpret_cast<const T*>(&v[u]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) see(head + (c + u * kThreads) * VEC + k, e[k]);
      }
  }
  const unsigned tail = head + chunks * VEC + threadIdx.x;
  if (tail < s.count) see(tail, p[tail]);
}

// Gather the rank keys of a bin into the leader's list. Returns their number.
template <typename T>
__device__ __forceinline__ unsigned gather(cg::cluster_group& cluster, State* st, State* lead,
                                           const Slice<T>& s, float top, int bin) {
  if (cluster.block_rank() == 0 && threadIdx.x == 0) st->listed = 0;
  cluster.sync();
#pragma unroll 4
  for (unsigned i = threadIdx.x; i < s.count; i += kThreads) {
    const float x = s.at(i);
    if (bin_of(x, top) == bin) {
      const unsigned at = atomicAdd(&lead->listed, 1u);
      if (at < kList) lead->list[at] = rank_key(x, s.first + i);
    }
  }
  cluster.sync();
  return lead->listed;
}

// The cut inside `bin`: the rank key of its need-th token or, with need == 0, of
// the first at which the weight from the bin's top reaches goal. `upto` gets the
// weight up to and with the cut. All CTAs of the cluster call it together; the
// results are valid in all.
template <typename T>
__device__ __forceinline__ void cut_bin(cg::cluster_group& cluster, State* st, State* lead,
                                        const Slice<T>& s, float top, int bin, unsigned need, u64 goal,
                                        u64& cut, u64& upto) {
  const unsigned n = gather(cluster, st, lead, s, top, bin);
  if (n <= kList) {
    if (cluster.block_rank() == 0) {
      for (unsigned i = threadIdx.x; i < n; i += kThreads) {
        const u64 mine = st->list[i];
        unsigned rank = 0;
#pragma unroll 4
        for (unsigned j = 0; j < n; ++j) rank += st->list[j] > mine;
        st->sorted[rank] = mine;
      }
      __syncthreads();
      const unsigned a = 2 * threadIdx.x, b = a + 1;
      const u64 wa = a < n ? weight_of(mass_of(x_of(st->sorted[a]), top)) : 0;
      const u64 wb = b < n ? weight_of(mass_of(x_of(st->sorted[b]), top)) : 0;
      const u64 before = block_before64(wa + wb, st->red);
      const u64 ua = before + wa, ub = ua + wb;
      if (a < n && (need ? a + 1 == need : before < goal && ua >= goal)) st->cut = st->sorted[a], st->goal = ua;
      if (b < n && (need ? b + 1 == need : ua < goal && ub >= goal)) st->cut = st->sorted[b], st->goal = ub;
    }
    cluster.sync();
    cut = lead->cut, upto = lead->goal;
    cluster.sync();  // before the leader's words are written again
    return;
  }
  // radix passes over the rank key, eight bits at a time, highest digit first
  u64 prefix = 0, above = 0;
  unsigned left = need;
#pragma unroll 1
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) st->wbin[i] = 0, st->cbin[i] = 0;
    cluster.sync();
    const u64 mask = shift == 56 ? 0 : ~0ull << (shift + 8);
#pragma unroll 1
    for (unsigned i = threadIdx.x; i < s.count; i += kThreads) {
      const float x = s.at(i);
      if (bin_of(x, top) != bin) continue;
      const u64 k = rank_key(x, s.first + i);
      if ((k ^ prefix) & mask) continue;
      const int d = (int)(k >> shift) & 255;
      atomicAdd(&lead->cbin[d], 1u);
      atomicAdd(&lead->wbin[d], weight_of(mass_of(x, top)));
    }
    cluster.sync();
    if (cluster.block_rank() == 0 && threadIdx.x == 0) {
      u64 w = above;
      unsigned c = 0;
      int d = 255;
      for (; d > 0; --d) {
        if (need ? c + st->cbin[d] >= left : w + st->wbin[d] >= goal) break;
        c += st->cbin[d], w += st->wbin[d];
      }
      st->cut = prefix | (u64)d << shift;
      st->need = left - c;
      st->goal = w;
      st->total = w + st->wbin[d];
    }
    cluster.sync();
    prefix = lead->cut, left = lead->need, above = lead->goal, upto = lead->total;
    cluster.sync();
  }
  cut = prefix;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ sy_sample_args a,
                                                             unsigned slice, bool resident) {
  extern __shared__ __align__(16) char smem[];
  State* st = reinterpret_cast<State*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank(), ctas = cluster.num_blocks();
  State* lead = cluster.map_shared_rank(st, 0);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long r = blockIdx.x / ctas;
  const unsigned V = (unsigned)a.vocab;
  const float temp = a.temperature ? a.temperature[r] : 1.f;
  const bool greedy = !(temp > 0.f);

  Slice<T> s;
  s.row = static_cast<const T*>(a.logits) + r * a.logits_row;
  s.first = min(V, rank * slice);
  s.count = min(V, (rank + 1) * slice) - s.first;
  s.x = resident ? reinterpret_cast<float*>(smem + sizeof(State)) : nullptr;
  s.inv_t = greedy ? 1.f : __fdiv_rn(1.f, temp);

  // the maximum and its lowest index
  float top;
  unsigned at;
  read_slice(s, top, at);
  if (at != 0xffffffffu) at += s.first;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float y = __shfl_xor_sync(kFull, top, o);
    const unsigned i = __shfl_xor_sync(kFull, at, o);
    if (y > top || (y == top && i < at)) top = y, at = i;
  }
  if (lane == 0) st->fred[warp] = top, st->ured[warp] = at;
  for (int i = tid; i < kBins; i += kThreads) st->wbin[i] = 0, st->cbin[i] = 0;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w)
      if (st->fred[w] > top || (st->fred[w] == top && st->ured[w] < at)) top = st->fred[w], at = st->ured[w];
    st->max_x = top, st->max_at = at;
  }
  cluster.sync();
  top = -INFINITY, at = 0xffffffffu;
  for (unsigned c = 0; c < ctas; ++c) {
    const State* o = cluster.map_shared_rank(st, c);
    if (o->max_x > top || (o->max_x == top && o->max_at < at)) top = o->max_x, at = o->max_at;
  }

  const long long k = greedy ? 1 : a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f;
  if (top == -INFINITY || k == 1) {
    // nothing to draw from, or one token: its share is the whole
    if (rank == 0 && tid == 0) {
      const bool none = top == -INFINITY;
      a.token[r] = none ? -1 : (long long)at;
      if (a.logprob) a.logprob[r] = none ? NAN : 0.f;
    }
    cluster.sync();  // the others may still be reading this CTA's maximum
    return;
  }

  u64 cut = 0;  // kept: rank keys from the cut on
  const bool by_count = k > 0 && k < V, by_weight = p < 1.f;
  if (by_count || by_weight) {
#pragma unroll 4
    for (unsigned i = tid; i < s.count; i += kThreads) {
      const float x = s.at(i);
      const int b = bin_of(x, top);
      if (b < kBins) {
        atomicAdd(&st->cbin[b], 1u);
        if (by_weight) atomicAdd(&st->wbin[b], weight_of(mass_of(x, top)));
      }
    }
    cluster.sync();
    if (rank) {
      for (int i = tid; i < kBins; i += kThreads)
        if (st->cbin[i]) {
          atomicAdd(&lead->cbin[i], st->cbin[i]);
          if (by_weight) atomicAdd(&lead->wbin[i], st->wbin[i]);
        }
    }
    cluster.sync();
    // The leader's threads have four bins each: counts and weights before them.
    constexpr int kEach = kBins / kThreads;
    u64 c_before = 0, w_before = 0, z = 0;
    if (rank == 0) {
      u64 c = 0, w = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) c += st->cbin[tid * kEach + i], w += st->wbin[tid * kEach + i];
      c_before = block_before64(c, st->red);
      w_before = block_before64(w, st->red);
      z = block_sum64(w, st->red);
      if (tid == 0) st->bin = kBins;
      __syncthreads();
      if (by_count) {
        u64 seen = c_before, weight = w_before;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int b = tid * kEach + i;
          if (seen < (u64)k && seen + st->cbin[b] >= (u64)k)
            st->bin = b, st->need = (unsigned)((u64)k - seen), st->goal = weight;
          seen += st->cbin[b], weight += st->wbin[b];
        }
      }
    }
    cluster.sync();
    int last = lead->bin;  // the bin that top_k cuts
    unsigned need = lead->need;
    u64 ahead = lead->goal;  // weight before it
    cluster.sync();
    if (last < kBins) {
      // cut_bin's radix passes use the first bins' words: keep the leader's copy
      u64 keep_w = 0;
      unsigned keep_c = 0;
      if (rank == 0 && tid < 256) keep_w = st->wbin[tid], keep_c = st->cbin[tid];
      u64 upto;
      cut_bin(cluster, st, lead, s, top, last, need, 0ull, cut, upto);
      __syncthreads();
      if (rank == 0 && tid < 256) st->wbin[tid] = keep_w, st->cbin[tid] = keep_c;
      __syncthreads();
      z = ahead + upto;
    }
    if (by_weight) {
      if (rank == 0) {
        const double g = ceil((double)fmaxf(p, 0.f) * (double)z);
        u64 goal = g < 1.0 ? 1ull : (u64)g;
        if (goal > z) goal = z;
        if (tid == 0) st->bin = last;
        __syncthreads();
        u64 weight = w_before;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int b = tid * kEach + i;
          if (b <= last && weight < goal && (weight + st->wbin[b] >= goal || b == last))
            st->bin = b, st->goal = goal - weight;
          weight += st->wbin[b];
        }
      }
      cluster.sync();
      const int bin = lead->bin;
      const u64 goal = lead->goal;
      cluster.sync();
      if (bin < kBins) {
        u64 upto, c;
        cut_bin(cluster, st, lead, s, top, bin, 0u, goal, c, upto);
        cut = c > cut ? c : cut;
      }
    }
  }

  // The kept weight, warp by warp in index order.
  const float min_p = fminf(a.min_p ? a.min_p[r] : 0.f, 1.f);
  const float low = cut ? x_of(cut) : -INFINITY;
  auto kept = [&](unsigned i) -> u64 {
    const float x = s.at(i);
    if (x < low || rank_key(x, s.first + i) < cut) return 0;
    const float e = mass_of(x, top);
    return e >= min_p ? weight_of(e) : 0;
  };
  const unsigned seg = (s.count + kThreads - 1) / kThreads * 32;  // a warp's part
  const unsigned w_first = min(s.count, warp * seg), w_last = min(s.count, w_first + seg);
  u64 sum = 0;
#pragma unroll 4
  for (unsigned i = w_first + lane; i < w_last; i += 32) sum += kept(i);
  sum = warp_sum64(sum);
  __syncthreads();
  if (lane == 0) st->red[warp] = sum;
  __syncthreads();
  u64 before = 0, mine = 0;
#pragma unroll 4
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += st->red[w];
    mine += st->red[w];
  }
  if (tid == 0) st->total = mine;
  cluster.sync();
  u64 total = 0;
  for (unsigned c = 0; c < ctas; ++c) {
    const u64 t = cluster.map_shared_rank(st, c)->total;
    if (c < rank) before += t;
    total += t;
  }
  const double g = floor((double)a.u[r] * (double)total);
  u64 aim = g > 0.0 ? (u64)g : 0ull;
  if (aim >= total) aim = total - 1;
  // the warp whose part holds the aim walks it
  if (before <= aim && aim < before + sum) {
#pragma unroll 1
    for (unsigned i0 = w_first; i0 < w_last; i0 += 32) {
      const u64 w = i0 + lane < w_last ? kept(i0 + lane) : 0;
      u64 upto = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 z = __shfl_up_sync(kFull, upto, o);
        if (lane >= o) upto += z;
      }
      upto += before;
      if (w && upto > aim && upto - w <= aim) {
        a.token[r] = s.first + i0 + lane;
        if (a.logprob) a.logprob[r] = logf(__fdiv_rn((float)w, (float)total));
      }
      before = __shfl_sync(kFull, upto, 31);
      if (before > aim) break;
    }
  }
  cluster.sync();  // no CTA ends while another reads its words
}

template <typename T>
cudaError_t launch_type(const sy_sample_args& a, cudaStream_t st) {
  // A CTA for every 4096 tokens up to 8: few rows gain by the latency, many rows
  // lose little (a slice of 512 threads x 8 values still covers a barrier).
  unsigned ctas = 1;
  while (ctas < kMaxCluster && (int64_t)ctas * 4096 < a.vocab) ctas *= 2;
  unsigned slice = (unsigned)((a.vocab + ctas - 1) / ctas);
  slice = (slice + 15) / 16 * 16;
  const bool resident = (int64_t)slice * 4 <= kMaxSlice;
  const size_t smem = sizeof(State) + (resident ? (size_t)slice * 4 : 0);
  cudaError_t e = raise_smem_limit(sample_kernel<T>, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, a, slice, resident);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

int64_t sample_workspace(const sy_sample_args&, const ServingDev&) { return 0; }

cudaError_t launch_sample(const sy_sample_args& a, const ServingDev&, cudaStream_t st) {
  switch (a.dtype) {
    case SY_BF16:
      return launch_type<__nv_bfloat16>(a, st);
    case SY_F16:
      return launch_type<__half>(a, st);
    case SY_F32:
      return launch_type<float>(a, st);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace sy

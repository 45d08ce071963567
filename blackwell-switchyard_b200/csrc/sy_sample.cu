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
// 28.4 are zero), at first only in the quarter next to the maximum, as a cut
// rarely lies deeper and most tokens do; the bin that holds the cut has a few tokens, as a rule, which
// are gathered and ranked by comparing all pairs. A bin with more than kList of
// them (ties, flat rows) is cut by eight radix passes over the rank keys instead.
// The draw then adds the kept weights in index order: CTAs, warps, lanes.
//
// The row's bytes are the floor for many rows (256 x 131071 fp32: 20.5 us at the
// measured copy rate; 246 us, 44 % of the issue slots and about 37 rows in flight);
// for few rows (1 x 32000: 18 us) it is a chain of cluster barriers: three without
// top_k and top_p or for one token, seven with one of them or with both cuts in
// one bin, nine with the cuts in two, two more where the bins next to the maximum
// do not hold the cut, and 32 for each cut made by radix passes.
// A remote shared-memory read costs as much as a barrier, so CTAs push what others
// need (maxima, sums, the leader's verdicts) ahead of the barrier and read locally.
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
constexpr int kNear = 512;                           // bins filled at first: 7.1 below the maximum
constexpr int64_t kMaxSlice = 128 * 1024;            // bytes of a slice in shared memory

// What the leader found, pushed to every CTA.
struct Verdict {
  u64 cut;        // kept so far: rank keys from here on
  u64 goal;       // weight of p_bin from its top to the cut
  int k_bin;      // the bin that top_k cuts, kBins if none
  int p_bin;      // the bin that top_p cuts, kBins if none (or not known before top_k's cut)
  unsigned need;  // tokens of k_bin up to the cut
  int enough;     // the bins filled so far hold the cuts
};

struct State {
  u64 wbin[kBins];       // weight per bin
  unsigned cbin[kBins];  // tokens per bin
  u64 list[kList];       // rank keys of this CTA's tokens in the bin that is cut
  u64 all[kList];        // leader: every CTA's
  u64 sorted[kList];     // also the radix passes' bins
  unsigned listed[2];
  Verdict verdict;
  // one per CTA of the cluster, pushed
  float max_x[kMaxCluster];
  unsigned max_at[kMaxCluster];
  u64 sums[kMaxCluster], kept[kMaxCluster];
  u64 found, upto;       // leader: a cut, and the weight up to and with it
  u64 goal_above;        // leader: weight above the radix passes' prefix
  unsigned left;
  u64 red[2][kWarps];
  float fred[kWarps];
  unsigned ured[kWarps];
};

constexpr size_t kStateBytes = (sizeof(State) + 15) / 16 * 16;

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
// rint(2^40 e). Below 2^23 adding 2^23 rounds to a whole number and leaves it in
// the low bits; from there on the float is whole and its mantissa is shifted. (The
// 64-bit conversion instruction has a small fraction of this rate.)
__device__ __forceinline__ u64 weight_of(float e) {
  const float y = __fmul_rn(e, 1099511627776.f);
  if (y < 8388608.f) return __float_as_uint(__fadd_rn(y, 8388608.f)) - 0x4b000000u;
  const unsigned b = __float_as_uint(y);
  return (u64)((b & 0x7fffffu) | 0x800000u) << ((b >> 23) - 150u);
}
// Add to a 64-bit sum in shared memory by 32-bit atomics, which the hardware has:
// whoever wraps the low word carries.
__device__ __forceinline__ void add_weight(u64* sum, u64 w) {
  unsigned* word = reinterpret_cast<unsigned*>(sum);
  const unsigned lo = (unsigned)w, old = atomicAdd(word, lo);
  const unsigned hi = (unsigned)(w >> 32) + (old + lo < old ? 1u : 0u);
  if (hi) atomicAdd(word + 1, hi);
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
// Exclusive prefixes over the block of two values at a time; `all` gets the totals.
__device__ __forceinline__ void block_before(const u64 (&x)[2], u64 (&before)[2], u64 (&all)[2],
                                             u64 (*red)[kWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 y[2] = {x[0], x[1]};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 a = __shfl_up_sync(kFull, y[0], o), b = __shfl_up_sync(kFull, y[1], o);
    if (lane >= o) y[0] += a, y[1] += b;
  }
  __syncthreads();
  if (lane == 31) red[0][warp] = y[0], red[1][warp] = y[1];
  __syncthreads();
  // each half of the warp adds up one value's sums
  u64 w = red[lane >> 4][lane & 15];
  u64 mine = (lane & 15) < warp ? w : 0;
#pragma unroll
  for (int o = 8; o; o >>= 1) w += __shfl_xor_sync(kFull, w, o), mine += __shfl_xor_sync(kFull, mine, o);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    all[i] = __shfl_sync(kFull, w, 16 * i);
    before[i] = y[i] - x[i] + __shfl_sync(kFull, mine, 16 * i);
  }
}
static_assert(kWarps == 16, "block_before: one value's sums are half a warp's lanes");

template <typename T, bool Resident>
struct Slice {
  const T* row;
  float* x;  // Resident: the slice's scaled logits in shared memory
  unsigned first, count;
  float inv_t;
  __device__ __forceinline__ float scaled(T v) const {
    const float y = __fmul_rn(Dt<T>::to_f(v), inv_t);
    return y == y ? y : -INFINITY;
  }
  __device__ __forceinline__ float at(unsigned i) const {
    return Resident ? x[i] : scaled(row[first + i]);
  }
};

// Read the slice and return its maximum; x goes to shared memory.
template <typename T, bool Resident>
__device__ __forceinline__ float read_slice(Slice<T, Resident>& s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  float top = -INFINITY;
  const T* p = s.row + s.first;
  // to the first 16-byte boundary, then whole chunks, four in flight, then the rest
  const unsigned head =
      min(s.count, (unsigned)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (unsigned)sizeof(T));
  s.x += (4 - head) & 3;  // so that the chunks' values are stored 16 bytes at a time
  auto see = [&](unsigned i) {
    const float y = s.scaled(p[i]);
    if (Resident) s.x[i] = y;
    top = fmaxf(top, y);
  };
  if (threadIdx.x < head) see(threadIdx.x);
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
        float y[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) y[k] = s.scaled(e[k]), top = fmaxf(top, y[k]);
        if (Resident)
#pragma unroll
          for (int k = 0; k < VEC; k += 4)
            *reinterpret_cast<float4*>(s.x + head + (c + u * kThreads) * VEC + k) =
                make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]);
      }
  }
  const unsigned tail = head + chunks * VEC + threadIdx.x;
  if (tail < s.count) see(tail);
  return top;
}

// The cut inside a bin from its gathered rank keys: the need-th or, with need == 0,
// the first at which the weight from the bin's top reaches goal. The leader's block
// only; the results are st->found and st->upto, valid after the block's barrier here.
__device__ __forceinline__ void rank_list(State* st, const u64* list, unsigned n, unsigned need, u64 goal,
                                          float top) {
  for (unsigned i = threadIdx.x; i < n; i += kThreads) {
    const u64 mine = list[i];
    unsigned rank = 0;
#pragma unroll 4
    for (unsigned j = 0; j < n; ++j) rank += list[j] > mine;
    st->sorted[rank] = mine;
  }
  __syncthreads();
  const unsigned a = 2 * threadIdx.x, b = a + 1;
  const u64 wa = a < n ? weight_of(mass_of(x_of(st->sorted[a]), top)) : 0;
  const u64 wb = b < n ? weight_of(mass_of(x_of(st->sorted[b]), top)) : 0;
  const u64 x[2] = {wa + wb, 0};
  u64 before[2], all[2];
  block_before(x, before, all, st->red);
  const u64 ua = before[0] + wa, ub = ua + wb;
  if (a < n && (need ? a + 1 == need : before[0] < goal && ua >= goal)) st->found = st->sorted[a], st->upto = ua;
  if (b < n && (need ? b + 1 == need : ua < goal && ub >= goal)) st->found = st->sorted[b], st->upto = ub;
  __syncthreads();
}

// The same for a bin with too many tokens for a list: eight radix passes over the
// rank keys, highest digit first, by the whole cluster into the leader's bins.
template <typename T, bool Resident>
__device__ __noinline__ void radix_cut(State* st, const Slice<T, Resident>& s, float top, int bin, unsigned need,
                                       u64 goal) {
  cg::cluster_group cluster = cg::this_cluster();
  const bool leads = cluster.block_rank() == 0;
  State* lead = cluster.map_shared_rank(st, 0);
  u64* wsum = lead->sorted;
  unsigned* csum = reinterpret_cast<unsigned*>(lead->sorted + 256);
  u64 prefix = 0, above = 0;
  unsigned left = need;
#pragma unroll 1
  for (int shift = 56; shift >= 0; shift -= 8) {
    if (leads)
      for (int i = threadIdx.x; i < 256; i += kThreads) wsum[i] = 0, csum[i] = 0;
    cluster.sync();
    const u64 mask = shift == 56 ? 0 : ~0ull << (shift + 8);
#pragma unroll 1
    for (unsigned i = threadIdx.x; i < s.count; i += kThreads) {
      const float x = s.at(i);
      if (bin_of(x, top) != bin) continue;
      const u64 k = rank_key(x, s.first + i);
      if ((k ^ prefix) & mask) continue;
      const int d = (int)(k >> shift) & 255;
      atomicAdd(&csum[d], 1u);
      atomicAdd(&wsum[d], weight_of(mass_of(x, top)));
    }
    cluster.sync();
    if (leads && threadIdx.x == 0) {
      u64 w = above;
      unsigned c = 0;
      int d = 255;
#pragma unroll 1
      for (; d > 0; --d) {
        if (need ? c + csum[d] >= left : w + wsum[d] >= goal) break;
        c += csum[d], w += wsum[d];
      }
      st->found = prefix | (u64)d << shift;
      st->left = left - c;
      st->goal_above = w;
      st->upto = w + wsum[d];
    }
    cluster.sync();
    prefix = lead->found, left = lead->left, above = lead->goal_above;
    cluster.sync();
  }
}

template <typename T, bool Resident>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ sy_sample_args a,
                                                             unsigned slice) {
  extern __shared__ __align__(16) char smem[];
  State* st = reinterpret_cast<State*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank(), ctas = cluster.num_blocks();
  const bool leads = rank == 0;
  State* lead = cluster.map_shared_rank(st, 0);
  // A CTA's shared memory may only be written from another once it is known to
  // run: all arrive here and wait before the first push, with the slice's read
  // in between.
  cluster.barrier_arrive();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long r = blockIdx.x / ctas;
  const unsigned V = (unsigned)a.vocab;
  const float temp = a.temperature ? a.temperature[r] : 1.f;
  const bool greedy = !(temp > 0.f);
  const long long k = greedy ? 1 : a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f;
  const float min_p = fminf(a.min_p ? a.min_p[r] : 0.f, 1.f);
  const float u = a.u[r];
  const bool by_count = k > 0 && k < V, by_weight = p < 1.f;

  Slice<T, Resident> s;
  s.row = static_cast<const T*>(a.logits) + r * a.logits_row;
  s.first = min(V, rank * slice);
  s.count = min(V, (rank + 1) * slice) - s.first;
  s.x = reinterpret_cast<float*>(smem + kStateBytes);
  s.inv_t = greedy ? 1.f : __fdiv_rn(1.f, temp);

  float top = warp_max(read_slice(s));
  if (lane == 0) st->fred[warp] = top;
  for (int i = tid; i < kBins; i += kThreads) st->wbin[i] = 0, st->cbin[i] = 0;
  if (tid < 2) st->listed[tid] = 0;
  __syncthreads();
  cluster.barrier_wait();
  if (warp == 0) {
    top = warp_max(st->fred[lane & 15]);
    if (lane < ctas) cluster.map_shared_rank(st, lane)->max_x[rank] = top;
  }
  cluster.sync();
  top = warp_max(lane < ctas ? st->max_x[lane] : -INFINITY);

  if (top == -INFINITY || k == 1) {
    // nothing to draw from, or one token, the first with the maximum: its share is the whole
    unsigned at = 0xffffffffu;
    if (top > -INFINITY)
#pragma unroll 4
      for (unsigned i = tid; i < s.count; i += kThreads)
        if (s.at(i) == top) at = min(at, s.first + i);
    at = __reduce_min_sync(kFull, at);
    if (lane == 0) st->ured[warp] = at;
    __syncthreads();
    if (warp == 0) {
      at = __reduce_min_sync(kFull, st->ured[lane & 15]);
      if (lane == 0) lead->max_at[rank] = at;
    }
    cluster.sync();  // nothing remote is touched after it
    if (leads && warp == 0) {
      at = __reduce_min_sync(kFull, lane < ctas ? st->max_at[lane] : 0xffffffffu);
      if (lane == 0) {
        const bool none = top == -INFINITY;
        a.token[r] = none ? -1 : (long long)at;
        if (a.logprob) a.logprob[r] = none ? NAN : 0.f;
      }
    }
    return;
  }

  u64 cut = 0;  // kept: rank keys from the cut on
  const float slack = fabsf(top) * 1e-6f;  // covers the rounding of max - x
  if (by_count || by_weight) {
    // Fill bins [b0, b1) and bring the cluster's together in the leader's; the
    // first time also add up all weights.
    auto fill = [&](int b0, int b1) {
      u64 sum = 0;
      // what no bin of these and (the first time) no sum wants goes by fast
      const float far = b0 == 0 && by_weight ? kSpan : b1 / kBinsPer;
      const float low = top < INFINITY ? top - far * 1.001f - slack : top;
#pragma unroll 4
      for (unsigned i = tid; i < s.count; i += kThreads) {
        const float x = s.at(i);
        if (x < low) continue;
        const u64 w = by_weight ? weight_of(mass_of(x, top)) : 0;
        if (b0 == 0) sum += w;
        const int b = bin_of(x, top);
        if (b < b0 || b >= b1) continue;
        if (by_count) atomicAdd(&st->cbin[b], 1u);
        if (by_weight) add_weight(&st->wbin[b], w);
      }
      if (b0 == 0) {
        const u64 x[2] = {sum, 0};
        u64 before[2], all[2];
        block_before(x, before, all, st->red);
        if (tid == 0) lead->sums[rank] = all[0];
      }
      cluster.sync();
      if (leads) {
#pragma unroll 1
        for (int b = b0 + tid; b < b1; b += kThreads) {
          u64 w[kMaxCluster];
          unsigned c[kMaxCluster];
#pragma unroll
          for (unsigned o = 1; o < kMaxCluster; ++o) {
            const State* other = cluster.map_shared_rank(st, o < ctas ? o : 0);
            w[o] = o < ctas ? other->wbin[b] : 0, c[o] = o < ctas ? other->cbin[b] : 0;
          }
          w[0] = st->wbin[b], c[0] = st->cbin[b];
#pragma unroll
          for (unsigned o = 1; o < kMaxCluster; ++o) w[0] += w[o], c[0] += c[o];
          st->wbin[b] = w[0], st->cbin[b] = c[0];
        }
        __syncthreads();
      }
    };
    // The leader's threads have four bins each; tokens and weight before them.
    constexpr int kEach = kBins / kThreads;
    u64 before[2], z = 0;
    auto p_of_z = [&]() -> u64 {
      const double g = ceil((double)fmaxf(p, 0.f) * (double)z);
      return g < 1.0 ? 1ull : min((u64)g, z);
    };
    // The bin where the weight reaches p of z (the last one allowed at the latest).
    auto find_weight = [&](int last) {
      const u64 goal = p_of_z();
      u64 weight = before[1];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int b = tid * kEach + i;
        if (b <= last && weight < goal && (weight + st->wbin[b] >= goal || b == last))
          st->verdict.p_bin = b, st->verdict.goal = goal - weight;
        weight += st->wbin[b];
      }
    };
    auto push_verdict = [&] {  // leader: to every CTA
      __syncthreads();
      constexpr int kWords = sizeof(Verdict) / 4;
      if (tid < kWords * (int)(ctas - 1))
        reinterpret_cast<unsigned*>(&cluster.map_shared_rank(st, 1 + tid / kWords)->verdict)[tid % kWords] =
            reinterpret_cast<unsigned*>(&st->verdict)[tid % kWords];
    };
    u64 ahead = 0;  // leader: weight before top_k's bin
    auto judge = [&](bool all_filled) {
      u64 x[2] = {0, 0}, sums[2];
#pragma unroll
      for (int i = 0; i < kEach; ++i) x[0] += st->cbin[tid * kEach + i], x[1] += st->wbin[tid * kEach + i];
      block_before(x, before, sums, st->red);
      z = lane < ctas ? st->sums[lane] : 0;
      z = warp_sum64(z);
      // enough, if k tokens were counted, or the weight that p asks for at most
      // (in whole numbers: a sum beyond 2^53 rounds up to a goal that it does not reach)
      const bool enough = all_filled || (by_count ? sums[0] >= (u64)k : sums[1] >= p_of_z());
      if (tid == 0) {
        st->verdict.enough = enough;
        st->verdict.k_bin = st->verdict.p_bin = kBins;
        st->verdict.cut = 0;
      }
      __syncthreads();
      if (enough && by_count) {
        u64 seen = before[0], weight = before[1];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int b = tid * kEach + i;
          if (seen < (u64)k && seen + st->cbin[b] >= (u64)k)
            st->verdict.k_bin = b, st->verdict.need = (unsigned)((u64)k - seen), st->upto = weight;
          seen += st->cbin[b], weight += st->wbin[b];
        }
        __syncthreads();
        ahead = st->upto;
      }
      if (enough && by_weight && st->verdict.k_bin == kBins) find_weight(kBins);
      push_verdict();
    };
    fill(0, kNear);
    if (leads) judge(false);
    cluster.sync();
    if (!st->verdict.enough) {
      fill(kNear, kBins);
      if (leads) judge(true);
      cluster.sync();
    }
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      const int bin = which ? st->verdict.p_bin : st->verdict.k_bin;
      if (bin == kBins) continue;
      const unsigned need = which ? 0u : st->verdict.need;
      const u64 goal = which ? st->verdict.goal : 0ull;
      // gather the bin's rank keys; a little beyond its ends tells the rest off
      // without the bin's arithmetic
      const float lo = top < INFINITY ? top - (bin + 1) / kBinsPer * 1.001f - slack : top;
      const float hi = top < INFINITY ? top - bin / kBinsPer * 0.999f + slack : top;
#pragma unroll 4
      for (unsigned i = tid; i < s.count; i += kThreads) {
        const float x = s.at(i);
        if (x >= lo && x <= hi && bin_of(x, top) == bin) {
          const unsigned n = atomicAdd(&st->listed[which], 1u);
          if (n < kList) st->list[n] = rank_key(x, s.first + i);
        }
      }
      cluster.sync();
      const unsigned got = lane < ctas ? cluster.map_shared_rank(st, lane)->listed[which] : 0;
      unsigned upto_got = got;
#pragma unroll
      for (int o = 1; o < kMaxCluster; o <<= 1) {
        const unsigned y = __shfl_up_sync(kFull, upto_got, o);
        if (lane >= o) upto_got += y;
      }
      const unsigned n = __shfl_sync(kFull, upto_got, kMaxCluster - 1);
      if (leads && n <= kList) {  // a warp or two per CTA bring the lists together
        const unsigned from = warp % kMaxCluster;
        const unsigned count = __shfl_sync(kFull, got, from), to = __shfl_sync(kFull, upto_got, from) - count;
        for (unsigned i = lane + warp / kMaxCluster * 32; i < count; i += kThreads / kMaxCluster)
          st->all[to + i] = cluster.map_shared_rank(st, from)->list[i];
        __syncthreads();
      }
      if (n > kList) radix_cut(st, s, top, bin, need, goal);
      if (leads) {
        if (n <= kList) rank_list(st, st->all, n, need, goal, top);
        const u64 found = st->found, upto = st->upto;
        __syncthreads();
        if (tid == 0) {
          if (found > st->verdict.cut) st->verdict.cut = found;
          st->verdict.p_bin = kBins;
        }
        if (which == 0 && by_weight) {
          z = ahead + upto;
          __syncthreads();
          find_weight(bin);
          __syncthreads();
          if (st->verdict.p_bin == bin && n <= kList) {  // the same bin: its list is here
            const u64 rest = st->verdict.goal;
            __syncthreads();
            rank_list(st, st->all, n, 0u, rest, top);
            if (tid == 0) {
              if (st->found > st->verdict.cut) st->verdict.cut = st->found;
              st->verdict.p_bin = kBins;
            }
          }
        }
        push_verdict();
      }
      cluster.sync();
    }
    cut = st->verdict.cut;
  }

  // The kept weight, warp by warp in index order.
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
  const u64 x[2] = {lane == 0 ? sum : 0, 0};
  u64 ahead[2], all[2];
  block_before(x, ahead, all, st->red);
  if (tid < (int)ctas) cluster.map_shared_rank(st, tid)->kept[rank] = all[0];
  cluster.sync();  // the last one: nothing remote is touched after it
  u64 total = lane < ctas ? st->kept[lane] : 0;
  u64 before = lane < rank ? total : 0;
  total = warp_sum64(total);
  before = warp_sum64(before) + __shfl_sync(kFull, ahead[0], 0);
  const double g = floor((double)u * (double)total);
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
        const u64 y = __shfl_up_sync(kFull, upto, o);
        if (lane >= o) upto += y;
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
  const size_t smem = kStateBytes + (resident ? (size_t)slice * 4 + 16 : 0);
  auto* kern = resident ? sample_kernel<T, true> : sample_kernel<T, false>;
  cudaError_t e = raise_smem_limit(kern, smem);
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
  e = cudaLaunchKernelEx(&cfg, kern, a, slice);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

cudaError_t launch_sample(const sy_sample_args& a, cudaStream_t st) {
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

// sy_sample.cu -- one token a row from logits and given random numbers.
//
// Weights are whole numbers (units of 2^-40 of the largest), so sums are exact
// whatever their order. One block per row. The rank of a token is decided by
// (key, index): key is x as an order-preserving 32-bit number, so a set of the
// highest ranks is "every key above t, and the first c of those equal to t".
// top_k and top_p each find such a (t, c) by three radix passes over the keys
// (11 + 11 + 10 bits) that count, or sum weights, per digit.
#include <cmath>

#include "sy_common.cuh"
#include "sy_launch.cuh"
#include "sy_serving.cuh"

namespace sy {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 2048;
using u64 = unsigned long long;

// x of element i: the scaled logit, NaN as -inf
template <typename T>
__device__ __forceinline__ float scaled(const T* row, long long i, float inv_t) {
  const float x = __fmul_rn(Dt<T>::to_f(row[i]), inv_t);
  return x == x ? x : -INFINITY;
}
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);  // -0 ranks with +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// exp(x - top), 1 where x is the maximum (infinities included)
__device__ __forceinline__ float mass_of(float x, float top) {
  return x == top ? 1.f : expf(__fsub_rn(x, top));
}
__device__ __forceinline__ u64 weight_of(float e) {
  return (u64)__float2ull_rn(__fmul_rn(e, 1099511627776.f));
}

template <typename V>
__device__ V block_sum(V x, V* scratch) {
  __syncthreads();
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
  __syncthreads();
  V s = 0;
  for (int w = 0; w < kThreads / 32; ++w) s += scratch[w];
  return s;
}

// inclusive scan over the block; *total gets the sum
template <typename V>
__device__ V block_scan(V x, V* scratch, V* total) {
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(kFull, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  V before = 0, all = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += scratch[w];
    all += scratch[w];
  }
  *total = all;
  return x + before;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_row_kernel(const sy_sample_args a) {
  __shared__ u64 bins[kBins];
  __shared__ u64 scratch[kThreads / 32];
  __shared__ float fscratch[kThreads / 32];
  __shared__ u64 found[2];  // digit, what is left of the goal inside it
  __shared__ long long answer;
  const long long r = blockIdx.x, V = a.vocab;
  const T* row = static_cast<const T*>(a.logits) + r * a.logits_row;
  const float temp = a.temperature ? a.temperature[r] : 1.f;
  const bool greedy = !(temp > 0.f);
  const float inv_t = greedy ? 1.f : __fdiv_rn(1.f, temp);
  float top = -INFINITY;
  for (long long i = threadIdx.x; i < V; i += kThreads) top = fmaxf(top, scaled(row, i, inv_t));
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) fscratch[threadIdx.x >> 5] = top;
  if (threadIdx.x == 0) answer = V;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, fscratch[w]);
  if (top == -INFINITY) {
    if (threadIdx.x == 0) {
      a.token[r] = -1;
      if (a.logprob) a.logprob[r] = NAN;
    }
    return;
  }
  // kept so far: keys above `edge`, and the first `ties` equal to it
  unsigned edge = 0;
  u64 ties = ~0ull;
  // what counts: the number of tokens (stage 0, top_k) or their weight (stage 1, top_p)
  long long k = greedy ? 1 : (a.top_k ? a.top_k[r] : 0);
  const float p = a.top_p ? a.top_p[r] : 1.f;
  for (int stage = 0; stage < 2; ++stage) {
    u64 goal;
    if (stage == 0) {
      if (k <= 0 || k >= V) continue;
      goal = (u64)k;
    } else {
      if (!(p < 1.f)) continue;
      u64 z = 0;
      for (long long i = threadIdx.x; i < V; i += kThreads) {
        const float x = scaled(row, i, inv_t);
        if (key_of(x) > edge) z += weight_of(mass_of(x, top));
      }
      z = block_sum(z, scratch);
      if (ties != ~0ull) {
        const unsigned b = edge & 0x80000000u ? edge ^ 0x80000000u : ~edge;
        z += ties * weight_of(mass_of(__uint_as_float(b), top));
      }
      const double g = ceil((double)fmaxf(p, 0.f) * (double)z);
      goal = g < 1.0 ? 1ull : (u64)g;
      if (goal > z) goal = z;
    }
    // the key at which the running total from the highest key down reaches goal
    unsigned prefix = 0;
    u64 left = goal;
    const int shift[3] = {21, 10, 0}, width[3] = {11, 11, 10};
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = threadIdx.x; i < kBins; i += kThreads) bins[i] = 0;
      __syncthreads();
      for (long long i = threadIdx.x; i < V; i += kThreads) {
        const float x = scaled(row, i, inv_t);
        const unsigned key = key_of(x);
        const bool match =
            pass == 0 || (key >> (shift[pass] + width[pass])) == (prefix >> (shift[pass] + width[pass]));
        if (!match) continue;
        const u64 w = stage == 0 ? 1ull : weight_of(mass_of(x, top));
        if (w) atomicAdd(&bins[(key >> shift[pass]) & ((1u << width[pass]) - 1)], w);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        u64 sum = 0;
        int digit = (1 << width[pass]) - 1;
        for (; digit > 0; --digit) {
          if (sum + bins[digit] >= left) break;
          sum += bins[digit];
        }
        found[0] = (u64)digit;
        found[1] = left - sum;
      }
      __syncthreads();
      prefix |= (unsigned)found[0] << shift[pass];
      left = found[1];
      __syncthreads();
    }
    const unsigned b = prefix & 0x80000000u ? prefix ^ 0x80000000u : ~prefix;
    u64 c = left;
    if (stage == 1) {
      const u64 w = weight_of(mass_of(__uint_as_float(b), top));
      c = w ? (left + w - 1) / w : ~0ull;
    }
    if (prefix > edge || (prefix == edge && c < ties)) edge = prefix, ties = c;
  }
  const float min_p = fminf(a.min_p ? a.min_p[r] : 0.f, 1.f);
  // two sweeps in index order: the kept total, then the draw
  u64 goal = 0, total = 0;
  for (int sweep = 0; sweep < 2; ++sweep) {
    u64 seen = 0, before = 0;
    for (long long base = 0; base < V; base += kThreads) {
      const long long i = base + threadIdx.x;
      const float x = i < V ? scaled(row, i, inv_t) : -INFINITY;
      const unsigned key = key_of(x);
      u64 tied = 0;
      u64 rank = 0;
      if (ties != ~0ull) rank = block_scan<u64>(i < V && key == edge, scratch, &tied);
      const bool in = i < V && (key > edge || (key == edge && (ties == ~0ull || before + rank <= ties)));
      before += tied;
      const float e = mass_of(x, top);
      const u64 w = in && e >= min_p ? weight_of(e) : 0;
      u64 part = 0;
      const u64 upto = seen + block_scan<u64>(w, scratch, &part);
      if (sweep == 1 && w && upto > goal && upto - w <= goal) {
        answer = i;
        if (a.logprob) a.logprob[r] = logf(__fdiv_rn((float)w, (float)total));
      }
      seen += part;
      if (sweep == 1 && seen > goal) break;
    }
    if (sweep == 0) {
      total = seen;
      const double g = floor((double)a.u[r] * (double)total);
      goal = g > 0.0 ? (u64)g : 0ull;
      if (goal >= total) goal = total - 1;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) a.token[r] = answer;
}

}  // namespace

int64_t sample_workspace(const sy_sample_args&, const ServingDev&) { return 0; }

cudaError_t launch_sample(const sy_sample_args& a, const ServingDev&, cudaStream_t st) {
  const dim3 grid((unsigned)a.rows);
  switch (a.dtype) {
    case SY_BF16:
      return launch_smem(sample_row_kernel<__nv_bfloat16>, grid, kThreads, 0, st, a);
    case SY_F16:
      return launch_smem(sample_row_kernel<__half>, grid, kThreads, 0, st, a);
    case SY_F32:
      return launch_smem(sample_row_kernel<float>, grid, kThreads, 0, st, a);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace sy

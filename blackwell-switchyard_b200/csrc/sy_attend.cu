// sy_attend.cu -- attention over a shared prefix and over each sequence's own
// pages.
//
// One block per output row (sequence, query token, head): its warps take the
// row's keys in turn, each with a running maximum and sum (an online softmax),
// and the warps' states are merged once at the end. All of it in fp32.
#include <cmath>

#include "sy_common.cuh"
#include "sy_launch.cuh"
#include "sy_serving.cuh"

namespace sy {
namespace {

constexpr int kWarps = 8;

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) attend_row_kernel(const sy_attend_args a) {
  __shared__ float sm_m[kWarps], sm_l[kWarps], sm_o[kWarps][128];
  const int hq = (int)a.q_heads, d = (int)a.head_dim;
  const long long r = blockIdx.x;
  const int h = (int)(r % hq);
  const int t = (int)(r / hq % a.q_len);
  const long long b = r / hq / a.q_len;
  const int kh = h / (hq / (int)a.kv_heads);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long len = a.kv_lens[b];
  const long long room = a.table_width * a.page_size;
  if (len > room || len < 0) {
    if (threadIdx.x == 0) record_device_error(kDevErrBadIndex);
    len = len < 0 ? 0 : room;
  }
  long long own = len - a.q_len + t + 1;
  if (own < 0) own = 0;
  const long long keys = a.prefix_len + own;
  const T* q = static_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + h * a.q_h;
  float qf[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int i = 0; i < 4; ++i)
    qf[i] = lane + 32 * i < d ? Dt<T>::to_f(q[lane + 32 * i]) * a.scale : 0.f;
  for (long long j = warp; j < keys; j += kWarps) {
    const bool shared = j < a.prefix_len;
    const long long i = shared ? j : j - a.prefix_len;
    const long long slot = i / a.page_size, row = i % a.page_size;
    const long long page =
        shared ? a.prefix_pages[slot] : a.page_table[b * a.table_row + slot];
    if (page < 0 || page >= a.pages) {
      if (lane == 0) record_device_error(kDevErrBadIndex);
      continue;
    }
    const T* k = static_cast<const T*>(a.k_cache) + page * a.kc_page + kh * a.kc_head + row * a.kc_row;
    const T* v = static_cast<const T*>(a.v_cache) + page * a.vc_page + kh * a.vc_head + row * a.vc_row;
    float s = 0.f, vf[4];
    for (int c = 0; c < 4; ++c) {
      const bool on = lane + 32 * c < d;
      s += qf[c] * (on ? Dt<T>::to_f(k[lane + 32 * c]) : 0.f);
      vf[c] = on ? Dt<T>::to_f(v[lane + 32 * c]) : 0.f;
    }
    s = warp_sum(s);
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : expf(m - top);
    const float p = top == -INFINITY ? 0.f : expf(s - top);
    m = top;
    l = l * keep + p;
    for (int c = 0; c < 4; ++c) o[c] = o[c] * keep + p * vf[c];
  }
  if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
  for (int c = 0; c < 4; ++c) sm_o[warp][lane + 32 * c] = o[c];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w]);
  for (int w = 0; w < kWarps; ++w)
    if (sm_m[w] != -INFINITY) total += sm_l[w] * expf(sm_m[w] - top);
  for (int c = threadIdx.x; c < d; c += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < kWarps; ++w)
      if (sm_m[w] != -INFINITY) x += sm_o[w][c] * expf(sm_m[w] - top);
    static_cast<T*>(a.out)[r * d + c] = Dt<T>::from_f(total > 0.f ? x / total : 0.f);
  }
  if (a.lse && threadIdx.x == 0) a.lse[r] = total > 0.f ? top + logf(total) : -INFINITY;
}

}  // namespace

int64_t attend_workspace(const sy_attend_args&, const ServingDev&) { return 0; }

cudaError_t launch_attend(const sy_attend_args& a, const ServingDev&, cudaStream_t st) {
  const dim3 grid((unsigned)(a.batch * a.q_len * a.q_heads));
  if (a.dtype == SY_BF16)
    return launch_smem(attend_row_kernel<__nv_bfloat16>, grid, 32 * kWarps, 0, st, a);
  return launch_smem(attend_row_kernel<__half>, grid, 32 * kWarps, 0, st, a);
}

}  // namespace sy

// sy_append.cu -- rotate new queries and keys, write new keys and values into
// the pages of a cache: one pass, one launch.
//
// Per element pair of a rotated half (x1, x2 = x[i], x[i + h]):
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s
// in fp32, rounded once. Bytes: every row read once and written once; 3 flops
// per element, so memory bounds it (for few tokens: the launch).
//
// One block per token, a "lane group" of L threads per head row: lane c < h/VEC
// turns chunk c against chunk c + h/VEC, the lanes after it copy what is not
// rotated, and a value row is copied by all L lanes. VEC is the widest access
// (16 bytes down to one element) that divides the halves, the strides and the
// addresses. The token's cos and sin rows come from L1 after the first head.
// 8192 tokens of 16 + 16 heads of 128 in bf16 take 51 us, 0.62 of the measured
// copy rate: the blocks are short, and what is in flight falls off between them.
// A single token takes 5.4 us, which is the launch and four dependent loads.
#include "sy_common.cuh"
#include "sy_launch.cuh"
#include "sy_serving.cuh"

namespace sy {
namespace {

template <typename T, int VEC>
struct Vec {
  static_assert(sizeof(T) * VEC <= 16, "one access");
  union {
    T e[VEC];
    uint4 q;
    uint2 d;
    uint32_t w;
    uint16_t h;
  };
  __device__ Vec() {}
  __device__ __forceinline__ void load(const T* p) {
    constexpr int B = sizeof(T) * VEC;
    if constexpr (B == 16)
      q = __ldg(reinterpret_cast<const uint4*>(p));
    else if constexpr (B == 8)
      d = __ldg(reinterpret_cast<const uint2*>(p));
    else if constexpr (B == 4)
      w = __ldg(reinterpret_cast<const uint32_t*>(p));
    else
      h = __ldg(reinterpret_cast<const uint16_t*>(p));
  }
  __device__ __forceinline__ void store(T* p) const {
    constexpr int B = sizeof(T) * VEC;
    if constexpr (B == 16)
      *reinterpret_cast<uint4*>(p) = q;
    else if constexpr (B == 8)
      *reinterpret_cast<uint2*>(p) = d;
    else if constexpr (B == 4)
      *reinterpret_cast<uint32_t*>(p) = w;
    else
      *reinterpret_cast<uint16_t*>(p) = h;
  }
};

// VEC floats of a row of cos or sin
template <int VEC>
__device__ __forceinline__ void load_angles(const float* p, bool aligned, float* x) {
  if constexpr (VEC % 4 == 0) {
    if (aligned) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p + i));
        x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = __ldg(p + i);
}

// Six blocks an SM: without the bound the compiler takes 80 registers and three fit.
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 6)
    append_kernel(const __grid_constant__ sy_append_kv_args a, int lanes, bool angles16) {
  const long long t = blockIdx.x;
  const int h = a.positions ? (int)a.rot_half : 0, d = (int)a.head_dim;
  const int group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const int groups = blockDim.x / lanes;
  long long slot = a.slots[t];
  const long long pos = h ? a.positions[t] : 0;
  const bool bad_pos = h && (pos < 0 || pos >= a.rope_len);
  const bool bad_slot = slot >= a.pages * a.page_size;
  if (bad_pos || bad_slot) {
    // not followed: the token's cache rows stay as they were, and its q is zero if
    // the position was outside (rotated as ever if only the slot was)
    if (threadIdx.x == 0) record_device_error(kDevErrBadIndex);
    slot = -1;
  }
  const int nq = (int)a.q_heads, nk = (int)a.kv_heads;
  if (bad_pos) {
    T* q = static_cast<T*>(a.q_out) + t * nq * (long long)d;
    for (int i = threadIdx.x; i < nq * d; i += blockDim.x) q[i] = Dt<T>::from_f(0.f);
    return;
  }
  const float* cs = a.cos + pos * a.rope_row;
  const float* sn = a.sin + pos * a.rope_row;
  long long page = 0, row = 0;
  if (slot >> 32) {
    if (slot > 0) page = slot / a.page_size, row = slot - page * a.page_size;
  } else {  // a 64-bit division costs as much as the rest of the kernel
    page = (unsigned)slot / (unsigned)a.page_size, row = (unsigned)slot - (unsigned)page * (unsigned)a.page_size;
  }
  const int pairs = h / VEC;
  const int rows = slot < 0 ? nq : nq + 2 * nk;
  if (group >= groups) return;
  for (int r = group; r < rows; r += groups) {
    const T* src;
    T* dst;
    int turned = pairs;
    if (r < nq) {
      src = static_cast<const T*>(a.q) + t * a.q_tok + r * a.q_head;
      dst = static_cast<T*>(a.q_out) + (t * nq + r) * (long long)d;
    } else if (r < nq + nk) {
      const int j = r - nq;
      src = static_cast<const T*>(a.k) + t * a.k_tok + j * a.k_head;
      dst = static_cast<T*>(a.k_cache) + page * a.kc_page + j * a.kc_head + row * a.kc_row;
    } else {
      const int j = r - nq - nk;
      src = static_cast<const T*>(a.v) + t * a.v_tok + j * a.v_head;
      dst = static_cast<T*>(a.v_cache) + page * a.vc_page + j * a.vc_head + row * a.vc_row;
      turned = 0;
    }
    for (int c = lane; c < turned; c += lanes) {
      Vec<T, VEC> x1, x2;
      x1.load(src + c * VEC);
      x2.load(src + c * VEC + h);
      float co[VEC], si[VEC];
      load_angles<VEC>(cs + c * VEC, angles16, co);
      load_angles<VEC>(sn + c * VEC, angles16, si);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float u = Dt<T>::to_f(x1.e[i]), w = Dt<T>::to_f(x2.e[i]);
        x1.e[i] = Dt<T>::from_f(__fsub_rn(__fmul_rn(u, co[i]), __fmul_rn(w, si[i])));
        x2.e[i] = Dt<T>::from_f(__fadd_rn(__fmul_rn(w, co[i]), __fmul_rn(u, si[i])));
      }
      x1.store(dst + c * VEC);
      x2.store(dst + c * VEC + h);
    }
    for (int c = 2 * turned + lane; c < d / VEC; c += lanes) {
      Vec<T, VEC> x;
      x.load(src + c * VEC);
      x.store(dst + c * VEC);
    }
  }
}

template <typename T, int VEC>
cudaError_t launch_vec(const sy_append_kv_args& a, cudaStream_t st) {
  const int h = a.positions ? (int)a.rot_half : 0;
  int lanes = h / VEC + (int)(a.head_dim - 2 * h) / VEC;
  if (lanes > 256) lanes = 256;
  const bool angles16 = ((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) & 15) == 0 &&
                        a.rope_row % 4 == 0;
  return launch_smem(append_kernel<T, VEC>, dim3((unsigned)a.tokens), dim3(256), 0, st, a, lanes, angles16);
}

template <typename T>
cudaError_t launch_type(const sy_append_kv_args& a, cudaStream_t st) {
  // the widest access that every row start, half and row length allows
  int64_t bytes = a.head_dim * (int64_t)sizeof(T);
  auto fold = [&](int64_t x) { bytes |= x * (int64_t)sizeof(T); };
  if (a.positions) fold(a.rot_half);
  if (a.q_heads) fold(a.q_tok), fold(a.q_head);
  fold(a.k_tok), fold(a.k_head), fold(a.v_tok), fold(a.v_head);
  fold(a.kc_page), fold(a.kc_head), fold(a.kc_row);
  fold(a.vc_page), fold(a.vc_head), fold(a.vc_row);
  const void* ptrs[] = {a.q, a.k, a.v, a.q_out, a.k_cache, a.v_cache};
  for (const void* p : ptrs) bytes |= (int64_t)reinterpret_cast<uintptr_t>(p);
  constexpr int E = (int)sizeof(T);
  if (bytes % 16 == 0) return launch_vec<T, 16 / E>(a, st);
  if (bytes % 8 == 0) return launch_vec<T, 8 / E>(a, st);
  if (bytes % 4 == 0) return launch_vec<T, 4 / E>(a, st);
  if constexpr (E == 2) return launch_vec<T, 1>(a, st);
  return cudaErrorMisalignedAddress;
}

}  // namespace

cudaError_t launch_append(const sy_append_kv_args& a, cudaStream_t st) {
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

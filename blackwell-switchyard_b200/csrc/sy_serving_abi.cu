// sy_serving_abi.cu -- the serving entry points of include/switchyard_b200.h:
// argument checks and dispatch. Nothing here allocates device memory or throws.
#include <cstdint>

#include "sy_launch.cuh"
#include "sy_serving.cuh"

namespace sy {
namespace {

// Sizes stay far below what the kernels' 64-bit index arithmetic can hold.
constexpr int64_t kMaxCount = int64_t(1) << 31;

cudaError_t serving_dev(ServingDev* d) {
  cudaError_t e = cudaGetDevice(&d->device);
  if (e != cudaSuccess) return e;
  return cudaDeviceGetAttribute(&d->sms, cudaDevAttrMultiProcessorCount, d->device);
}

bool known_dtype(int d) { return d == SY_BF16 || d == SY_F16 || d == SY_F32; }
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool in(int64_t x, int64_t lo, int64_t hi) { return x >= lo && x <= hi; }

int check_append(const sy_append_kv_args* a) {
  if (!a) return SY_ERR_ARG;
  if (!known_dtype(a->dtype)) return SY_ERR_DTYPE;
  if (!in(a->tokens, 0, kMaxCount - 1) || !in(a->q_heads, 0, 1 << 16) ||
      !in(a->kv_heads, 1, 1 << 16) || !in(a->head_dim, 1, 1 << 12))
    return SY_ERR_ARG;
  if (!in(a->page_size, 1, kMaxCount) || !in(a->pages, 0, kMaxCount)) return SY_ERR_ARG;
  if (a->tokens == 0) return SY_OK;
  if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->slots) return SY_ERR_ARG;
  if (a->q_heads > 0 && (!a->q || !a->q_out)) return SY_ERR_ARG;
  if (a->positions) {
    if (!a->cos || !a->sin || !in(a->rot_half, 1, a->head_dim / 2) ||
        !in(a->rope_len, 1, kMaxCount) || a->rope_row < a->rot_half)
      return SY_ERR_ARG;
  }
  return SY_OK;
}

int check_attend(const sy_attend_args* a, bool pointers) {
  if (!a) return SY_ERR_ARG;
  if (!known_dtype(a->dtype)) return SY_ERR_DTYPE;
  if (a->dtype == SY_F32) return SY_ERR_UNSUPPORTED;
  if (!in(a->batch, 0, 1 << 20) || !in(a->q_len, 0, 1 << 24) || !in(a->kv_heads, 1, 1 << 12) ||
      !in(a->q_heads, 1, 1 << 12) || !in(a->head_dim, 1, 1 << 12))
    return SY_ERR_ARG;
  if (a->q_heads % a->kv_heads != 0) return SY_ERR_ARG;
  if (a->head_dim % 8 != 0 || a->head_dim > 128 || a->page_size % 8 != 0)
    return SY_ERR_UNSUPPORTED;
  if (!in(a->page_size, 8, 1 << 20) || !in(a->pages, 0, kMaxCount - 1) ||
      !in(a->table_width, 0, kMaxCount - 1) || !in(a->prefix_len, 0, kMaxCount - 1))
    return SY_ERR_ARG;
  if (a->table_width * a->page_size >= kMaxCount) return SY_ERR_ARG;
  if (a->batch * a->q_len >= kMaxCount / a->q_heads) return SY_ERR_ARG;
  // the kernels multiply by scale * log2(e), which has to be finite too
  if (!(a->scale > 0.f) || a->scale > 2.35e38f) return SY_ERR_ARG;
  if (!pointers || a->batch == 0 || a->q_len == 0) return SY_OK;
  if (!a->q || !a->out || !a->kv_lens) return SY_ERR_ARG;
  if (a->prefix_len > 0 && !a->prefix_pages) return SY_ERR_ARG;
  if (a->table_width > 0 && !a->page_table) return SY_ERR_ARG;
  if ((a->table_width > 0 || a->prefix_len > 0) && a->pages > 0 && (!a->k_cache || !a->v_cache))
    return SY_ERR_ARG;
  if (!al16(a->q) || !al16(a->k_cache) || !al16(a->v_cache) || !al16(a->out)) return SY_ERR_ARG;
  // {length, stride} of each axis; that of one element may carry any stride
  const int64_t axes[][2] = {{a->batch, a->q_b},         {a->q_len, a->q_t},        {a->q_heads, a->q_h},
                             {a->pages, a->kc_page},     {a->kv_heads, a->kc_head}, {a->page_size, a->kc_row},
                             {a->pages, a->vc_page},     {a->kv_heads, a->vc_head}, {a->page_size, a->vc_row}};
  for (const auto& x : axes)
    if (x[0] > 1 && (x[1] < 0 || x[1] % 8 != 0 || x[1] > (int64_t(1) << 38))) return SY_ERR_ARG;
  // the kernel counts the start of a query row in 32 bits, in units of 16 bytes
  int64_t reach = 0;
  for (int i = 0; i < 3; ++i) {
    const int64_t more = axes[i][0] - 1, step = axes[i][1];
    if (more > 0 && step > (int64_t(1) << 35) / more) return SY_ERR_UNSUPPORTED;
    reach += more > 0 ? more * step : 0;
  }
  if (reach >= int64_t(1) << 35) return SY_ERR_UNSUPPORTED;
  return SY_OK;
}

int check_sample(const sy_sample_args* a, bool pointers) {
  if (!a) return SY_ERR_ARG;
  if (!known_dtype(a->dtype)) return SY_ERR_DTYPE;
  // 2^22 weights of at most 2^40 sum below 2^62
  if (!in(a->rows, 0, 1 << 24) || !in(a->vocab, 1, 1 << 22)) return SY_ERR_ARG;
  if (a->rows > 1 && a->logits_row < a->vocab) return SY_ERR_ARG;
  if (!pointers || a->rows == 0) return SY_OK;
  if (!a->logits || !a->u || !a->token) return SY_ERR_ARG;
  return SY_OK;
}

}  // namespace
}  // namespace sy

extern "C" {

int sy_append_kv(const sy_append_kv_args* args, sy_stream_t stream) {
  const int st = sy::check_append(args);
  if (st != SY_OK || args->tokens == 0) return st;
  return sy::cuda_error_status(sy::launch_append(*args, static_cast<cudaStream_t>(stream)),
                       "sy_append_kv");
}

int64_t sy_attend_workspace(const sy_attend_args* args) {
  const int st = sy::check_attend(args, false);
  if (st != SY_OK) return -st;
  if (args->batch == 0 || args->q_len == 0) return 0;
  sy::ServingDev dev;
  const cudaError_t e = sy::serving_dev(&dev);
  if (e != cudaSuccess) return -sy::cuda_error_status(e, "sy_attend_workspace");
  return sy::attend_workspace(*args, dev);
}

int sy_attend(const sy_attend_args* args, sy_stream_t stream) {
  const int st = sy::check_attend(args, true);
  if (st != SY_OK || args->batch == 0 || args->q_len == 0) return st;
  sy::ServingDev dev;
  const cudaError_t e = sy::serving_dev(&dev);
  if (e != cudaSuccess) return sy::cuda_error_status(e, "sy_attend");
  const int64_t need = sy::attend_workspace(*args, dev);
  if (need < 0) return (int)-need;
  if (args->workspace_bytes < need ||
      (args->workspace_bytes > 0 && (!args->workspace || !sy::al16(args->workspace))))
    return SY_ERR_ARG;
  return sy::cuda_error_status(sy::launch_attend(*args, dev, static_cast<cudaStream_t>(stream)),
                       "sy_attend");
}

int64_t sy_sample_workspace(const sy_sample_args* args) {
  const int st = sy::check_sample(args, false);
  return st == SY_OK ? 0 : -st;
}

int sy_sample(const sy_sample_args* args, sy_stream_t stream) {
  const int st = sy::check_sample(args, true);
  if (st != SY_OK || args->rows == 0) return st;
  return sy::cuda_error_status(sy::launch_sample(*args, static_cast<cudaStream_t>(stream)),
                               "sy_sample");
}

}  // extern "C"

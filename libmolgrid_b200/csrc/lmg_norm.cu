// Layer norm over the last dimension and its gradients.
#include "lmg_vectors.h"

namespace lmg {
namespace {

constexpr int THREADS = 128;

// the sum over the block, the same for all its threads
__device__ float block_sum(float v) {
  __shared__ float part[THREADS / 32];
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < THREADS / 32; i++) v += part[i];
  return v;
}

template <class T, class P>
__global__ void __launch_bounds__(THREADS) k_norm(Slots S, int width, const T* x, long long x_ld, const P* weight, const P* bias, float eps,
                                                  T* out, long long out_ld, float* stats) {
  wait_for_stream();
  const unsigned row = blockIdx.x;
  const T* in = x + (long long)row * x_ld;
  T* to = out + (long long)row * out_ld;
  if (!slot_filled(S, row)) {
    for (int c = threadIdx.x; c < width; c += THREADS) to[c] = from_float<T>(0.f);
    if (stats != nullptr && threadIdx.x < 2) stats[2ll * row + threadIdx.x] = 0.f;
    return;
  }
  float sum = 0.f;
  for (int c = threadIdx.x; c < width; c += THREADS) sum += to_float(in[c]);
  const float mean = block_sum(sum) / (float)width;
  sum = 0.f;
  for (int c = threadIdx.x; c < width; c += THREADS) {
    const float d = to_float(in[c]) - mean;
    sum += d * d;
  }
  const float q = 1.f / sqrtf(block_sum(sum) / (float)width + eps);
  for (int c = threadIdx.x; c < width; c += THREADS) {
    const float w = weight ? to_float(weight[c]) : 1.f, b = bias ? to_float(bias[c]) : 0.f;
    to[c] = from_float<T>((to_float(in[c]) - mean) * q * w + b);
  }
  if (stats != nullptr && threadIdx.x == 0) {
    stats[2ll * row] = mean;
    stats[2ll * row + 1] = q;
  }
}

template <class T, class P>
__global__ void __launch_bounds__(THREADS) k_norm_backward(Slots S, int width, const T* x, long long x_ld, const P* weight, const float* stats,
                                                           const T* diff, long long diff_ld, T* grad, long long grad_ld) {
  wait_for_stream();
  const unsigned row = blockIdx.x;
  const T* in = x + (long long)row * x_ld;
  const T* g = diff + (long long)row * diff_ld;
  T* to = grad + (long long)row * grad_ld;
  if (!slot_filled(S, row)) {
    for (int c = threadIdx.x; c < width; c += THREADS) to[c] = from_float<T>(0.f);
    return;
  }
  const float mean = stats[2ll * row], q = stats[2ll * row + 1];
  float s0 = 0.f, s1 = 0.f;
  for (int c = threadIdx.x; c < width; c += THREADS) {
    const float a = to_float(g[c]) * (weight ? to_float(weight[c]) : 1.f), h = (to_float(in[c]) - mean) * q;
    s0 += a;
    s1 += a * h;
  }
  s0 = block_sum(s0) / (float)width;
  s1 = block_sum(s1) / (float)width;
  for (int c = threadIdx.x; c < width; c += THREADS) {
    const float a = to_float(g[c]) * (weight ? to_float(weight[c]) : 1.f), h = (to_float(in[c]) - mean) * q;
    to[c] = from_float<T>(q * (a - s0 - h * s1));
  }
}

// a block per column sums over the rows
template <class T, class P>
__global__ void __launch_bounds__(THREADS) k_norm_weights(Slots S, const T* x, long long x_ld, const float* stats, const T* diff, long long diff_ld,
                                                          P* dweight, P* dbias) {
  wait_for_stream();
  const int c = blockIdx.x;
  float dw = 0.f, db = 0.f;
  for (unsigned r = threadIdx.x; r < S.rows; r += THREADS) {
    if (!slot_filled(S, r)) continue;
    const float g = to_float(diff[(long long)r * diff_ld + c]);
    dw += g * ((to_float(x[(long long)r * x_ld + c]) - stats[2ll * r]) * stats[2ll * r + 1]);
    db += g;
  }
  dw = block_sum(dw);
  db = block_sum(db);
  if (threadIdx.x == 0) {
    if (dweight) dweight[c] = from_float<P>(dw);
    if (dbias) dbias[c] = from_float<P>(db);
  }
}

// F(T, P) for the element types of vectors and parameters, which agree or the latter are float32
template <class F>
cudaError_t by_types(int type, int weight_type, F f) {
  if (type == LMG_FLOAT32) return f(float(), float());
  if (type == LMG_BFLOAT16) return weight_type == LMG_FLOAT32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
  return weight_type == LMG_FLOAT32 ? f(__half(), float()) : f(__half(), __half());
}

int check_weights(int type, int weight_type) {
  if (weight_type != type && weight_type != LMG_FLOAT32)
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "weights neither float32 nor of the vectors' type");
  return LMG_OK;
}

}  // namespace
}  // namespace lmg

extern "C" {

size_t lmg_vectors_workspace_bytes(int op, int rows, int ntypes, int width) {
  if (rows < 0 || ntypes < 0 || width < 0) return 0;
  return op == LMG_OP_EMBED_BACKWARD ? lmg::embed_backward_bytes((unsigned)rows, ntypes, width) : 256;
}

int lmg_layer_norm(const lmg_slots* rows, int width, const lmg_vectors* x, const void* weight, const void* bias, int weight_type,
                   float eps, const lmg_vectors* out, float* stats, void* stream) {
  using namespace lmg;
  int rc;
  if ((rc = check_slots(rows, width))) return rc;
  if (!(eps > 0.f)) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "eps must be positive");
  if (rows->batch == 0 || rows->max_atoms == 0 || width == 0) return LMG_OK;
  if ((rc = check_vectors(x, width, "input")) || (rc = check_vectors(out, width, "output"))) return rc;
  if (x->type != out->type) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "input and output differ in type");
  if ((rc = check_weights(x->type, weight_type))) return rc;
  const Slots S = to_slots(rows, 0);
  const cudaError_t e = by_types(x->type, weight_type, [&](auto t, auto p) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    return launch_early(k_norm<T, P>, dim3(S.rows), THREADS, 0, (cudaStream_t)stream, S, width, static_cast<const T*>(x->data), x->ld,
                        static_cast<const P*>(weight), static_cast<const P*>(bias), eps, static_cast<T*>(out->data), out->ld, stats);
  });
  if (e != cudaSuccess) return vectors_cuda(e, "layer norm");
  lmg_internal_count_launches(1);
  return LMG_OK;
}

int lmg_layer_norm_backward(const lmg_slots* rows, int width, const lmg_vectors* x, const void* weight, int weight_type,
                            const float* stats, const lmg_vectors* diff, const lmg_vectors* x_gradients, void* weight_gradients,
                            void* bias_gradients, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace lmg;
  int rc;
  if ((rc = check_slots(rows, width))) return rc;
  if (width == 0) return LMG_OK;
  const bool none = rows->batch == 0 || rows->max_atoms == 0;
  if (!none) {
    if ((rc = check_vectors(x, width, "input")) || (rc = check_vectors(diff, width, "diff")) ||
        (rc = check_vectors(x_gradients, width, "input gradients")))
      return rc;
    if (x->type != diff->type || x->type != x_gradients->type)
      return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "input, diff and input gradients differ in type");
    if ((rc = check_weights(x->type, weight_type))) return rc;
    if (stats == nullptr) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "stats missing memory");
  } else if (weight_type < LMG_FLOAT32 || weight_type > LMG_FLOAT16) {
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "weights of unknown element type");
  }
  const size_t need = lmg_vectors_workspace_bytes(LMG_OP_LAYER_NORM_BACKWARD, rows->batch * rows->max_atoms, 0, width);
  if (workspace == nullptr || workspace_bytes < need) return vectors_fail(LMG_ERR_WORKSPACE, "workspace too small for the gradients of a layer norm");
  const cudaStream_t st = (cudaStream_t)stream;
  if (none) {  // sums of nothing
    cudaError_t e = cudaSuccess;
    if (weight_gradients) e = cudaMemsetAsync(weight_gradients, 0, width * element_bytes(weight_type), st);
    if (e == cudaSuccess && bias_gradients) e = cudaMemsetAsync(bias_gradients, 0, width * element_bytes(weight_type), st);
    return e == cudaSuccess ? LMG_OK : vectors_cuda(e, "gradients of a layer norm");
  }
  const Slots S = to_slots(rows, 0);
  const cudaError_t e = by_types(x->type, weight_type, [&](auto t, auto p) {
    typedef decltype(t) T;
    typedef decltype(p) P;
    const T *xp = static_cast<const T*>(x->data), *gp = static_cast<const T*>(diff->data);
    cudaError_t e = cudaSuccess;
    if (weight_gradients || bias_gradients)
      e = launch_early(k_norm_weights<T, P>, dim3((unsigned)width), THREADS, 0, st, S, xp, x->ld, stats, gp, diff->ld, static_cast<P*>(weight_gradients),
                       static_cast<P*>(bias_gradients));
    if (e != cudaSuccess) return e;
    return launch_early(k_norm_backward<T, P>, dim3(S.rows), THREADS, 0, st, S, width, xp, x->ld, static_cast<const P*>(weight), stats, gp,
                        diff->ld, static_cast<T*>(x_gradients->data), x_gradients->ld);
  });
  if (e != cudaSuccess) return vectors_cuda(e, "gradients of a layer norm");
  lmg_internal_count_launches(weight_gradients || bias_gradients ? 2 : 1);
  return LMG_OK;
}

}  // extern "C"

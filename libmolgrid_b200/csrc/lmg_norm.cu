// Layer norm over the last dimension and its gradients.
#include "lmg_vectors.h"

namespace lmg {
namespace {

constexpr int VALUES = 8;                       // of a row that a thread holds in registers
constexpr int BLOCK = 256;                      // threads of a block whose rows each lie within a warp
constexpr int ROW_THREADS_MOST = 1024;          // of a row: 8192 columns
constexpr int WIDE = VALUES * ROW_THREADS_MOST;  // beyond it rows are read more than once (k_norm_wide, ...)

// A row's values over its `n` threads: VEC, 16 bytes a thread and turn, else an element a thread and turn, so that
// neighbouring threads always read neighbouring bytes.
template <class T, bool VEC>
struct Share {
  static constexpr int PER = VEC ? 16 / sizeof(T) : 1;
  static __device__ __forceinline__ int col(int thread, int n, int i) { return (thread + n * (i / PER)) * PER + i % PER; }
  static __device__ __forceinline__ void load(const T* row, int thread, int n, int width, float (&v)[VALUES]) {
#pragma unroll
    for (int k = 0; k < VALUES; k += PER) {
      const int c = col(thread, n, k);
      if (VEC && c + PER <= width) {
        const uint4 a = *reinterpret_cast<const uint4*>(row + c);
        const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < PER; i++) v[k + i] = to_float(e[i]);
      } else {
#pragma unroll
        for (int i = 0; i < PER; i++) v[k + i] = c + i < width ? to_float(row[c + i]) : 0.f;
      }
    }
  }
  static __device__ __forceinline__ void store(T* row, int thread, int n, int width, const float (&v)[VALUES]) {
#pragma unroll
    for (int k = 0; k < VALUES; k += PER) {
      const int c = col(thread, n, k);
      if (VEC && c + PER <= width) {
        uint4 a;
        T* e = reinterpret_cast<T*>(&a);
#pragma unroll
        for (int i = 0; i < PER; i++) e[i] = from_float<T>(v[k + i]);
        *reinterpret_cast<uint4*>(row + c) = a;
      } else {
#pragma unroll
        for (int i = 0; i < PER; i++)
          if (c + i < width) row[c + i] = from_float<T>(v[k + i]);
      }
    }
  }
};

// Sums over the threads of a row, the same for all of them: `n` lanes next to each other, or (SPAN) the whole block.  A block's
// sums take turns with two places in shared memory, so one barrier a sum is enough.
template <bool SPAN, int SUMS>
struct RowSum {
  float (*part)[SUMS][32];
  int n, turn = 0;
  __device__ __forceinline__ void operator()(float (&v)[SUMS]) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
      if (SPAN || o < n) {
#pragma unroll
        for (int s = 0; s < SUMS; s++) v[s] += __shfl_xor_sync(0xffffffffu, v[s], o);
      }
    if (SPAN) {
      const int lane = threadIdx.x & 31, warps = blockDim.x / 32;
      float (*p)[32] = part[turn];
      turn ^= 1;
      if (lane == 0) {
#pragma unroll
        for (int s = 0; s < SUMS; s++) p[s][threadIdx.x / 32] = v[s];
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < SUMS; s++) {
        v[s] = lane < warps ? p[s][lane] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) v[s] += __shfl_xor_sync(0xffffffffu, v[s], o);
      }
    }
  }
};

struct NormArgs {
  Slots S;
  int width, threads;  // threads of a row: a power of two up to 32, or the block
  unsigned tiles;      // of blockDim / threads rows
  float eps;
};

// Layer norm with the row in registers: mean, then the squares of what is left.  A block goes from row to row with its weights in
// registers and the next row's loads under way.
template <class T, class P, bool VEC, bool SPAN>
__global__ void __launch_bounds__(SPAN ? 1024 : BLOCK) k_norm(NormArgs A, const T* x, long long x_ld, const P* weight, const P* bias, T* out,
                                                              long long out_ld, float* stats) {
  typedef Share<T, VEC> Sh;
  __shared__ float part[2][1][32];
  const int n = SPAN ? blockDim.x : A.threads, thread = SPAN ? threadIdx.x : threadIdx.x & (n - 1);
  const unsigned rows = SPAN ? 1 : BLOCK / n, sub = SPAN ? 0 : threadIdx.x / n;
  RowSum<SPAN, 1> sum = {part, n};
  wait_for_stream();
  float w[VALUES], b[VALUES];
#pragma unroll
  for (int i = 0; i < VALUES; i++) {
    const int c = Sh::col(thread, n, i);
    w[i] = weight != nullptr && c < A.width ? to_float(weight[c]) : 1.f;
    b[i] = bias != nullptr && c < A.width ? to_float(bias[c]) : 0.f;
  }
  const float inv = 1.f / (float)A.width;
  float v[VALUES], next[VALUES];
  auto fetch = [&](unsigned tile, float (&to)[VALUES]) {
    const unsigned row = tile * rows + sub;
    const bool there = tile < A.tiles && row < A.S.rows && slot_filled(A.S, row);
    if (there) Sh::load(x + (long long)row * x_ld, thread, n, A.width, to);
    return there;
  };
  bool there = fetch(blockIdx.x, v);
  for (unsigned tile = blockIdx.x; tile < A.tiles; tile += gridDim.x) {
    const bool then = fetch(tile + gridDim.x, next);
    const unsigned row = tile * rows + sub;
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
      if (!there) v[i] = 0.f;
      s[0] += v[i];
    }
    sum(s);
    const float mean = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
      v[i] = Sh::col(thread, n, i) < A.width ? v[i] - mean : 0.f;
      s[0] += v[i] * v[i];
    }
    sum(s);
    const float q = 1.f / sqrtf(s[0] * inv + A.eps);
    if (row < A.S.rows) {
#pragma unroll
      for (int i = 0; i < VALUES; i++) v[i] = there ? v[i] * q * w[i] + b[i] : 0.f;
      Sh::store(out + (long long)row * out_ld, thread, n, A.width, v);
      if (stats != nullptr && thread == 0) reinterpret_cast<float2*>(stats)[row] = there ? make_float2(mean, q) : make_float2(0.f, 0.f);
    }
    there = then;
#pragma unroll
    for (int i = 0; i < VALUES; i++) v[i] = next[i];
  }
}

// dx = q (a - mean a - h mean(a h)) row by row, and with SUMS the sums over the block's rows of g h and g, which stay in the
// registers of the threads that hold their columns: parts[block][2][width].
template <class T, class P, bool VEC, bool SPAN, bool SUMS>
__global__ void __launch_bounds__(SPAN ? 1024 : BLOCK) k_norm_backward(NormArgs A, const T* x, long long x_ld, const P* weight, const float* stats,
                                                                       const T* diff, long long diff_ld, T* grad, long long grad_ld, float* parts) {
  typedef Share<T, VEC> Sh;
  __shared__ float part[2][2][32];
  const int n = SPAN ? blockDim.x : A.threads, thread = SPAN ? threadIdx.x : threadIdx.x & (n - 1);
  const unsigned rows = SPAN ? 1 : BLOCK / n, sub = SPAN ? 0 : threadIdx.x / n;
  RowSum<SPAN, 2> sum = {part, n};
  wait_for_stream();
  float w[VALUES], dw[VALUES] = {}, db[VALUES] = {};
#pragma unroll
  for (int i = 0; i < VALUES; i++) {
    const int c = Sh::col(thread, n, i);
    w[i] = weight != nullptr && c < A.width ? to_float(weight[c]) : 1.f;
  }
  const float inv = 1.f / (float)A.width;
  float v[VALUES], g[VALUES], next_v[VALUES], next_g[VALUES];
  float2 st, next_st;
  auto fetch = [&](unsigned tile, float (&to_v)[VALUES], float (&to_g)[VALUES], float2& to_st) {
    const unsigned row = tile * rows + sub;
    const bool there = tile < A.tiles && row < A.S.rows && slot_filled(A.S, row);
    if (there) {
      Sh::load(x + (long long)row * x_ld, thread, n, A.width, to_v);
      Sh::load(diff + (long long)row * diff_ld, thread, n, A.width, to_g);
      to_st = reinterpret_cast<const float2*>(stats)[row];
    }
    return there;
  };
  bool there = fetch(blockIdx.x, v, g, st);
  for (unsigned tile = blockIdx.x; tile < A.tiles; tile += gridDim.x) {
    const bool then = fetch(tile + gridDim.x, next_v, next_g, next_st);
    const unsigned row = tile * rows + sub;
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
      if (!there) v[i] = g[i] = 0.f;
      else v[i] = (v[i] - st.x) * st.y;
      if (SUMS) {
        dw[i] += g[i] * v[i];
        db[i] += g[i];
      }
      g[i] *= w[i];
      s[0] += g[i];
      s[1] += g[i] * v[i];
    }
    sum(s);
    const float s0 = s[0] * inv, s1 = s[1] * inv;
    if (row < A.S.rows) {
#pragma unroll
      for (int i = 0; i < VALUES; i++) v[i] = there ? st.y * (g[i] - s0 - v[i] * s1) : 0.f;
      Sh::store(grad + (long long)row * grad_ld, thread, n, A.width, v);
    }
    there = then;
    st = next_st;
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
      v[i] = next_v[i];
      g[i] = next_g[i];
    }
  }
  if (!SUMS) return;
  float* mine = parts + (size_t)blockIdx.x * 2 * A.width;
  if (SPAN) {
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
      const int c = Sh::col(thread, n, i);
      if (c < A.width) {
        mine[c] = dw[i];
        mine[A.width + c] = db[i];
      }
    }
  } else {
    // rows of a warp, then the warps
    __shared__ float all[2][BLOCK / 32][VALUES * 32];
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
      for (int o = 16; o >= n; o >>= 1) {
        dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
        db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
      }
      const int lane = threadIdx.x & 31;
      if (lane < n) {
        all[0][threadIdx.x / 32][Sh::col(lane, n, i)] = dw[i];
        all[1][threadIdx.x / 32][Sh::col(lane, n, i)] = db[i];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * VALUES * n; c += BLOCK) {
      const int which = c >= VALUES * n, at = c - which * VALUES * n;
      if (at >= A.width) continue;
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < BLOCK / 32; k++) t += all[which][k][at];
      mine[which * A.width + at] = t;
    }
  }
}

// the blocks' sums: 32 columns a block, 32 threads a column
template <class P>
__global__ void __launch_bounds__(1024) k_norm_sums(const float* parts, int n, int width, P* dweight, P* dbias) {
  __shared__ float s[32][33];
  wait_for_stream();
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x / 32;
  P* to = blockIdx.y ? dbias : dweight;
  if (to == nullptr) return;
  float sum = 0.f;
  if (c < width) {
    const float* p = parts + (size_t)blockIdx.y * width + c;
#pragma unroll 4
    for (int k = slice; k < n; k += 32) sum += p[(size_t)k * 2 * width];
  }
  s[slice][threadIdx.x & 31] = sum;
  __syncthreads();
  sum = s[threadIdx.x & 31][slice];  // a warp a column
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int col = blockIdx.x * 32 + slice;
  if ((threadIdx.x & 31) == 0 && col < width) to[col] = from_float<P>(sum);
}

// ---- rows of more than WIDE columns: a block a row, read again for each sum (from the L1, which holds a row of 200 KB) ----------------
constexpr int WIDE_THREADS = 1024;

template <class T, class P>
__global__ void __launch_bounds__(WIDE_THREADS) k_norm_wide(NormArgs A, const T* x, long long x_ld, const P* weight, const P* bias, T* out,
                                                            long long out_ld, float* stats) {
  __shared__ float part[2][1][32];
  RowSum<true, 1> sum = {part, WIDE_THREADS};
  wait_for_stream();
  const unsigned row = blockIdx.x;
  const T* in = x + (long long)row * x_ld;
  T* to = out + (long long)row * out_ld;
  if (!slot_filled(A.S, row)) {
    for (int c = threadIdx.x; c < A.width; c += WIDE_THREADS) to[c] = from_float<T>(0.f);
    if (stats != nullptr && threadIdx.x < 2) stats[2ll * row + threadIdx.x] = 0.f;
    return;
  }
  float s[1] = {0.f};
  for (int c = threadIdx.x; c < A.width; c += WIDE_THREADS) s[0] += to_float(in[c]);
  sum(s);
  const float mean = s[0] / (float)A.width;
  s[0] = 0.f;
  for (int c = threadIdx.x; c < A.width; c += WIDE_THREADS) {
    const float d = to_float(in[c]) - mean;
    s[0] += d * d;
  }
  sum(s);
  const float q = 1.f / sqrtf(s[0] / (float)A.width + A.eps);
  for (int c = threadIdx.x; c < A.width; c += WIDE_THREADS) {
    const float w = weight ? to_float(weight[c]) : 1.f, b = bias ? to_float(bias[c]) : 0.f;
    to[c] = from_float<T>((to_float(in[c]) - mean) * q * w + b);
  }
  if (stats != nullptr && threadIdx.x == 0) {
    stats[2ll * row] = mean;
    stats[2ll * row + 1] = q;
  }
}

template <class T, class P>
__global__ void __launch_bounds__(WIDE_THREADS) k_norm_backward_wide(NormArgs A, const T* x, long long x_ld, const P* weight, const float* stats,
                                                                     const T* diff, long long diff_ld, T* grad, long long grad_ld) {
  __shared__ float part[2][2][32];
  RowSum<true, 2> sum = {part, WIDE_THREADS};
  wait_for_stream();
  const unsigned row = blockIdx.x;
  const T* in = x + (long long)row * x_ld;
  const T* g = diff + (long long)row * diff_ld;
  T* to = grad + (long long)row * grad_ld;
  if (!slot_filled(A.S, row)) {
    for (int c = threadIdx.x; c < A.width; c += WIDE_THREADS) to[c] = from_float<T>(0.f);
    return;
  }
  const float mean = stats[2ll * row], q = stats[2ll * row + 1];
  float s[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < A.width; c += WIDE_THREADS) {
    const float a = to_float(g[c]) * (weight ? to_float(weight[c]) : 1.f), h = (to_float(in[c]) - mean) * q;
    s[0] += a;
    s[1] += a * h;
  }
  sum(s);
  const float s0 = s[0] / (float)A.width, s1 = s[1] / (float)A.width;
  for (int c = threadIdx.x; c < A.width; c += WIDE_THREADS) {
    const float a = to_float(g[c]) * (weight ? to_float(weight[c]) : 1.f), h = (to_float(in[c]) - mean) * q;
    to[c] = from_float<T>(q * (a - s0 - h * s1));
  }
}

// the sums over a block's share of the rows, 32 columns and 8 rows at a time; parts[blockIdx.y][2][width]
template <class T>
__global__ void __launch_bounds__(256) k_norm_weights_wide(NormArgs A, unsigned per, const T* x, long long x_ld, const float* stats, const T* diff,
                                                           long long diff_ld, float* parts) {
  __shared__ float s[2][8][32];
  wait_for_stream();
  const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, slice = threadIdx.x / 32;
  const unsigned begin = blockIdx.y * per, end = min(begin + per, A.S.rows);
  float dw = 0.f, db = 0.f;
  if (c < A.width)
    for (unsigned r = begin + slice; r < end; r += 8) {
      if (!slot_filled(A.S, r)) continue;
      const float g = to_float(diff[(long long)r * diff_ld + c]);
      dw += g * ((to_float(x[(long long)r * x_ld + c]) - stats[2ll * r]) * stats[2ll * r + 1]);
      db += g;
    }
  s[0][slice][lane] = dw;
  s[1][slice][lane] = db;
  __syncthreads();
  if (slice < 2 && c < A.width) {
    float t = 0.f;
    for (int k = 0; k < 8; k++) t += s[slice][k][lane];
    parts[((size_t)blockIdx.y * 2 + slice) * A.width + c] = t;
  }
}

// ---- the plan: a function of the sizes alone ------------------------------------------------------------------------------------
struct NormPlan {
  bool wide;
  int threads, block;      // of a row, of a block
  unsigned tiles, blocks;  // blocks: of the backward pass, whose sums are apart
  unsigned per;            // rows of a block of the wide sums
  size_t bytes;
};

NormPlan norm_plan(unsigned rows, int width) {
  NormPlan p = {};
  p.wide = width > WIDE;
  if (p.wide) {
    p.blocks = rows / 64 < 1 ? 1 : rows / 64 > 64 ? 64 : rows / 64;
    p.per = (rows + p.blocks - 1) / p.blocks;
  } else {
    p.threads = 1;
    while (p.threads < 32 && p.threads * VALUES < width) p.threads *= 2;
    if (p.threads * VALUES < width) p.threads = (width + VALUES * 32 - 1) / (VALUES * 32) * 32;
    p.block = p.threads > 32 ? p.threads : BLOCK;
    const unsigned per = p.threads > 32 ? 1 : BLOCK / p.threads;
    p.tiles = (rows + per - 1) / per;
    const unsigned resident = 148 * (unsigned)(1024 / p.block);
    p.blocks = p.tiles < resident ? p.tiles : resident;
  }
  p.bytes = 256 + (size_t)p.blocks * 2 * width * 4;
  return p;
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

int check_stats(const float* stats) {
  if (reinterpret_cast<uintptr_t>(stats) % 8 != 0) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "stats not aligned to 8 bytes");
  return LMG_OK;
}

}  // namespace
}  // namespace lmg

extern "C" {

size_t lmg_vectors_workspace_bytes(int op, int rows, int ntypes, int width) {
  if (rows < 0 || ntypes < 0 || width < 0) return 0;
  return op == LMG_OP_EMBED_BACKWARD ? lmg::embed_backward_bytes((unsigned)rows, ntypes, width) : lmg::norm_plan((unsigned)rows, width).bytes;
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
  if ((rc = check_weights(x->type, weight_type)) || (rc = check_stats(stats))) return rc;
  NormArgs A = {to_slots(rows, 0), width, 0, 0, eps};
  const NormPlan p = norm_plan(A.S.rows, width);
  A.threads = p.threads;
  A.tiles = p.tiles;
  const bool vec = rows_aligned(x) && rows_aligned(out);
  const cudaError_t e = by_types(x->type, weight_type, [&](auto t, auto q) {
    typedef decltype(t) T;
    typedef decltype(q) P;
    auto kernel = k_norm_wide<T, P>;
    if (!p.wide && p.threads > 32) kernel = vec ? k_norm<T, P, true, true> : k_norm<T, P, false, true>;
    else if (!p.wide) kernel = vec ? k_norm<T, P, true, false> : k_norm<T, P, false, false>;
    return launch_early(kernel, dim3(p.wide ? A.S.rows : p.blocks), p.wide ? WIDE_THREADS : p.block, 0, (cudaStream_t)stream, A,
                        static_cast<const T*>(x->data), x->ld, static_cast<const P*>(weight), static_cast<const P*>(bias),
                        static_cast<T*>(out->data), out->ld, stats);
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
    if ((rc = check_stats(stats))) return rc;
  } else if (weight_type < LMG_FLOAT32 || weight_type > LMG_FLOAT16) {
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "weights of unknown element type");
  }
  NormArgs A = {to_slots(rows, 0), width, 0, 0, 0.f};
  const NormPlan p = norm_plan(A.S.rows, width);
  A.threads = p.threads;
  A.tiles = p.tiles;
  if (workspace == nullptr || workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return vectors_fail(LMG_ERR_WORKSPACE, "workspace too small for the gradients of a layer norm, or off 16 bytes");
  const cudaStream_t st = (cudaStream_t)stream;
  if (none) {  // sums of nothing
    cudaError_t e = cudaSuccess;
    if (weight_gradients) e = cudaMemsetAsync(weight_gradients, 0, width * element_bytes(weight_type), st);
    if (e == cudaSuccess && bias_gradients) e = cudaMemsetAsync(bias_gradients, 0, width * element_bytes(weight_type), st);
    return e == cudaSuccess ? LMG_OK : vectors_cuda(e, "gradients of a layer norm");
  }
  const bool vec = rows_aligned(x) && rows_aligned(diff) && rows_aligned(x_gradients), sums = weight_gradients || bias_gradients;
  float* parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
  long launches = 0;
  const cudaError_t e = by_types(x->type, weight_type, [&](auto t, auto q) {
    typedef decltype(t) T;
    typedef decltype(q) P;
    const T *xp = static_cast<const T*>(x->data), *gp = static_cast<const T*>(diff->data);
    T* to = static_cast<T*>(x_gradients->data);
    cudaError_t e = cudaSuccess;
    if (p.wide && sums) {  // first: the gradients may take the place of diff
      e = launch_early(k_norm_weights_wide<T>, dim3((width + 31) / 32, p.blocks), 256, 0, st, A, p.per, xp, x->ld, stats, gp, diff->ld, parts);
      if (e != cudaSuccess) return e;
      launches++;
    }
    if (p.wide) {
      e = launch_early(k_norm_backward_wide<T, P>, dim3(A.S.rows), WIDE_THREADS, 0, st, A, xp, x->ld, static_cast<const P*>(weight), stats, gp,
                       diff->ld, to, x_gradients->ld);
    } else {
      auto kernel = k_norm_backward<T, P, false, false, false>;
      const int which = (vec ? 4 : 0) + (p.threads > 32 ? 2 : 0) + (sums ? 1 : 0);
      if (which == 1) kernel = k_norm_backward<T, P, false, false, true>;
      if (which == 2) kernel = k_norm_backward<T, P, false, true, false>;
      if (which == 3) kernel = k_norm_backward<T, P, false, true, true>;
      if (which == 4) kernel = k_norm_backward<T, P, true, false, false>;
      if (which == 5) kernel = k_norm_backward<T, P, true, false, true>;
      if (which == 6) kernel = k_norm_backward<T, P, true, true, false>;
      if (which == 7) kernel = k_norm_backward<T, P, true, true, true>;
      e = launch_early(kernel, dim3(p.blocks), p.block, 0, st, A, xp, x->ld, static_cast<const P*>(weight), stats, gp, diff->ld, to, x_gradients->ld,
                       parts);
    }
    if (e != cudaSuccess) return e;
    launches++;
    if (!sums) return e;
    launches++;
    return launch_early(k_norm_sums<P>, dim3((width + 31) / 32, 2), 1024, 0, st, parts, (int)p.blocks, width, static_cast<P*>(weight_gradients),
                        static_cast<P*>(bias_gradients));
  });
  lmg_internal_count_launches(launches);
  return e == cudaSuccess ? LMG_OK : vectors_cuda(e, "gradients of a layer norm");
}

}  // extern "C"

// Layer norm over the last dimension and its gradients.
#include "lmg_vectors.h"

namespace lmg {
namespace {

constexpr int BLOCK = 256;      // threads of a block whose rows each lie within a warp
constexpr int WIDE = 8192;      // columns; beyond it rows are read more than once (k_norm_wide, ...)
constexpr int MIDDLE = 2048;    // columns up to which a thread holds eight values of a row, sixteen beyond
// rows that are in use or on their way; both arrays of the widest rows fit an SM: 3 x 2 x 32 KB of float32, 4 x 2 x 16 KB of 16 bits
template <class T> constexpr int STAGES = sizeof(T) == 4 ? 3 : 4;

__device__ __forceinline__ void copy_async(unsigned to, const void* from, unsigned bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T> __device__ __forceinline__ Pair unpack(unsigned w);
template <> __device__ __forceinline__ Pair unpack<__nv_bfloat16>(unsigned w) { return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ Pair unpack<__half>(unsigned w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pair(f.x, f.y);
}
template <class T> __device__ __forceinline__ unsigned packed(Pair p);
template <> __device__ __forceinline__ unsigned packed<__nv_bfloat16>(Pair p) {
  float a, b;
  split(p, a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <> __device__ __forceinline__ unsigned packed<__half>(Pair p) {
  float a, b;
  split(p, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}

// A thread's VALUES values of the rows it works on, brought through shared memory by asynchronous copies of 16 bytes, so that rows under
// way take no registers.  VEC: rows begin on 16 bytes, a turn is 16 bytes a thread, and a thread copies what it
// reads itself and waits for no one.  Otherwise a turn is an element a thread; the row's threads copy the 16-byte pieces that
// the row lies in, from the one before its first value to its end, and wait for one another.  Neighbouring threads always
// touch neighbouring bytes.
template <class T, bool VEC, int VALUES>
struct Share {
  static constexpr int PER = VEC ? 16 / sizeof(T) : 1, COPIES = VALUES * sizeof(T) / 16;
  int thread, n, width;
  bool full;                // all its columns are the row's
  unsigned size[COPIES];    // VEC: bytes of its copies
  unsigned here, step;      // its first copy's place in a stage, from one to the next

  // bytes of a stage for a block of `block` threads, `n` a row
  static __host__ __device__ __forceinline__ unsigned bytes(unsigned block, unsigned n) { return block * COPIES * 16 + (VEC ? 0 : block / n * 32); }
  __device__ __forceinline__ int col(int i) const { return (thread + n * (i / PER)) * PER + i % PER; }
  __device__ __forceinline__ bool valid(int i) const { return col(i) < width; }

  __device__ __forceinline__ Share(int thread_, int n_, unsigned sub, int width_) : thread(thread_), n(n_), width(width_) {
    full = col(VALUES - 1) < width;
    here = VEC ? threadIdx.x * 16 : sub * (n * COPIES * 16 + 32);
    step = (VEC ? blockDim.x : n) * 16;
#pragma unroll
    for (int k = 0; k < COPIES; k++) {
      const int left = (width - col(k * PER)) * (int)sizeof(T);
      size[k] = left < 0 ? 0 : left < 16 ? left : 16;
    }
  }
  __device__ __forceinline__ void fetch(unsigned stage, const T* row) const {
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < COPIES; k++) copy_async(stage + here + k * step, size[k] ? row + (thread + n * k) * PER : row, size[k]);
    } else {
      const char* from = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(row) & ~(uintptr_t)15);
      const int all = (int)(reinterpret_cast<uintptr_t>(row) & 15) + width * (int)sizeof(T);
#pragma unroll
      for (int k = 0; k <= COPIES; k++) {
        const int at = (thread + n * k) * 16, left = all - at;
        if (left > 0) copy_async(stage + here + at, from + at, left < 16 ? left : 16);
      }
    }
  }
  __device__ __forceinline__ void take(const char* stage, const T* row, Pair (&v)[VALUES / 2]) const {
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < COPIES; k++) {  // what lies behind the row's end has been filled with zeros
        const uint4 a = *reinterpret_cast<const uint4*>(stage + here + k * step);
        if constexpr (sizeof(T) == 4) {
          v[2 * k] = pair(__uint_as_float(a.x), __uint_as_float(a.y));
          v[2 * k + 1] = pair(__uint_as_float(a.z), __uint_as_float(a.w));
        } else {
          v[4 * k] = unpack<T>(a.x), v[4 * k + 1] = unpack<T>(a.y), v[4 * k + 2] = unpack<T>(a.z), v[4 * k + 3] = unpack<T>(a.w);
        }
      }
    } else {
      const T* e = reinterpret_cast<const T*>(stage + here + (reinterpret_cast<uintptr_t>(row) & 15)) + thread;
      float f[VALUES];
      if (full) {
#pragma unroll
        for (int i = 0; i < VALUES; i++) f[i] = to_float(e[n * i]);
      } else {
#pragma unroll
        for (int i = 0; i < VALUES; i++) f[i] = valid(i) ? to_float(e[n * i]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < VALUES; i += 2) v[i / 2] = pair(f[i], f[i + 1]);
    }
  }
  __device__ __forceinline__ void store(T* row, const Pair (&v)[VALUES / 2]) const {
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < COPIES; k++) {
        T* to = row + (thread + n * k) * PER;
        uint4 a;
        if constexpr (sizeof(T) == 4) {
          float f[4];
          split(v[2 * k], f[0], f[1]);
          split(v[2 * k + 1], f[2], f[3]);
          a = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        } else {
          a = make_uint4(packed<T>(v[4 * k]), packed<T>(v[4 * k + 1]), packed<T>(v[4 * k + 2]), packed<T>(v[4 * k + 3]));
        }
        if (size[k] == 16) {
          *reinterpret_cast<uint4*>(to) = a;
        } else {
          const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
          for (int i = 0; i < PER; i++)
            if (i * sizeof(T) < size[k]) to[i] = e[i];
        }
      }
    } else {
      T* to = row + thread;
#pragma unroll
      for (int i = 0; i < VALUES; i += 2) {
        float f0, f1;
        split(v[i / 2], f0, f1);
        if (full || valid(i)) to[n * i] = from_float<T>(f0);
        if (full || valid(i + 1)) to[n * (i + 1)] = from_float<T>(f1);
      }
    }
  }
  // values that are not the row's to zero
  __device__ __forceinline__ void cut(Pair (&v)[VALUES / 2]) const {
    if (full) return;
#pragma unroll
    for (int i = 0; i < VALUES; i += 2) {
      float f0, f1;
      split(v[i / 2], f0, f1);
      v[i / 2] = pair(valid(i) ? f0 : 0.f, valid(i + 1) ? f1 : 0.f);
    }
  }
  template <class P>
  __device__ __forceinline__ void parameters(const P* p, float otherwise, Pair (&w)[VALUES / 2]) const {
#pragma unroll
    for (int i = 0; i < VALUES; i += 2)
      w[i / 2] = pair(p != nullptr && valid(i) ? to_float(p[col(i)]) : otherwise, p != nullptr && valid(i + 1) ? to_float(p[col(i + 1)]) : otherwise);
  }
};

// Sums over the threads of a row, the same for all of them: `n` lanes next to each other, or (SPAN) the whole block.  A block's
// sums take turns with two places in shared memory, so one barrier a sum is enough.
template <bool SPAN, int SUMS>
struct RowSum {
  float (*part)[SUMS][32];
  int n, turn = 0;
  __device__ __forceinline__ void lanes(float (&v)[SUMS], int from) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
      if (o < from) {
#pragma unroll
        for (int s = 0; s < SUMS; s++) v[s] += __shfl_xor_sync(0xffffffffu, v[s], o);
      }
  }
  __device__ __forceinline__ void operator()(float (&v)[SUMS]) {
    lanes(v, SPAN ? 32 : n);
    if (SPAN) {
      const int lane = threadIdx.x & 31, warps = blockDim.x / 32;
      float (*p)[32] = part[turn];
      turn ^= 1;
      if (lane == 0) {
#pragma unroll
        for (int s = 0; s < SUMS; s++) p[s][threadIdx.x / 32] = v[s];
      }
      __syncthreads();
      // each group of as many lanes as there are warps, rounded up to a power of two, adds up all of them
      const int at = lane & (n - 1);
#pragma unroll
      for (int s = 0; s < SUMS; s++) v[s] = at < warps ? p[s][at] : 0.f;
      lanes(v, n);
    }
  }
};

struct NormArgs {
  Slots S;
  int width, threads;  // threads of a row: a power of two up to 32, or the block
  int group;           // lanes that a sum goes over at the end: `threads`, or the block's warps rounded up to a power of two
  unsigned tiles;      // of blockDim / threads rows
  float eps;
};

// The rows of a block one after the other: which of them hold anything, looked up a turn before their copies begin.
struct Ahead {
  unsigned rows, sub, filled = 0;  // bit k: the row k turns from now
  int count = 0, place = 0;        // of the row whose copies come next
  __device__ __forceinline__ void look(const NormArgs& A, unsigned tile) {
    const unsigned row = tile * rows + sub;
    place = 0;
    count = tile < A.tiles && row < A.S.rows;
    if (A.S.n_atoms != nullptr && count != 0) {
      const unsigned b = A.S.by_n(row);
      place = (int)(row - b * A.S.n);
      count = A.S.n_atoms[b];
    }
  }
  __device__ __forceinline__ bool there() const { return place < count; }
};

// Layer norm with the row in registers: mean, then the squares of what is left.  A block goes from row to row with its weights in
// registers.  It is bound by what it issues where rows come from the L2: 16384 rows of 4096 bfloat16 took 91 us with eight values a thread,
// one at a time and checked against the row's end (307 instructions a warp and row).
template <class T, class P, bool VEC, bool SPAN, int VALUES>
__global__ void __launch_bounds__(VALUES == 16 ? 512 : BLOCK) k_norm(NormArgs A, const T* x, long long x_ld, const P* weight, const P* bias, T* out,
                                                                     long long out_ld, float* stats) {
  constexpr int H = VALUES / 2;
  extern __shared__ __align__(16) char ring[];
  __shared__ float part[2][1][32];
  const int n = SPAN ? blockDim.x : A.threads, thread = SPAN ? threadIdx.x : threadIdx.x & (n - 1);
  const unsigned rows = SPAN ? 1 : BLOCK / n, sub = SPAN ? 0 : threadIdx.x / n;
  const Share<T, VEC, VALUES> share(thread, n, sub, A.width);
  const unsigned stage = share.bytes(blockDim.x, n), ring_at = (unsigned)__cvta_generic_to_shared(ring);
  RowSum<SPAN, 1> sum = {part, A.group};
  wait_for_stream();
  Ahead ahead = {rows, sub};
  unsigned coming = blockIdx.x;  // the tile whose copies come next
  auto fetch = [&](int slot, int turn) {
    const bool there = ahead.there();
    if (there) share.fetch(ring_at + slot * stage, x + (long long)(coming * rows + sub) * x_ld);
    copies_end_group();
    ahead.filled |= (unsigned)there << turn;
    coming += gridDim.x;
    ahead.look(A, coming);
  };
  ahead.look(A, coming);
#pragma unroll
  for (int k = 0; k < STAGES<T> - 1; k++) fetch(k, k);
  Pair w[H], b[H];
  share.parameters(weight, 1.f, w);
  share.parameters(bias, 0.f, b);
  const float inv = 1.f / (float)A.width;
  int slot = 0;
  for (unsigned tile = blockIdx.x; tile < A.tiles; tile += gridDim.x) {
    if (!VEC && !SPAN) __syncwarp();  // the place that is filled next has been read
    fetch(slot == 0 ? STAGES<T> - 1 : slot - 1, STAGES<T> - 1);
    copies_but<STAGES<T> - 1>();
    if (!VEC) {
      if (SPAN) __syncthreads();
      else __syncwarp();
    }
    const bool there = ahead.filled & 1;
    ahead.filled >>= 1;
    const unsigned row = tile * rows + sub;
    Pair v[H];
    if (there) {
      share.take(ring + slot * stage, x + (long long)row * x_ld, v);
    } else {
#pragma unroll
      for (int k = 0; k < H; k++) v[k] = pair(0.f);
    }
    slot = slot == STAGES<T> - 1 ? 0 : slot + 1;
    float mean = 0.f, q = 0.f;
    if (!SPAN || there) {
      float s[1], t;
      Pair a = v[0];
#pragma unroll
      for (int k = 1; k < H; k++) a = add2(a, v[k]);
      split(a, s[0], t);
      s[0] += t;
      sum(s);
      mean = s[0] * inv;
#pragma unroll
      for (int k = 0; k < H; k++) v[k] = add2(v[k], pair(-mean));
      share.cut(v);
      a = mul2(v[0], v[0]);
#pragma unroll
      for (int k = 1; k < H; k++) a = fma2(v[k], v[k], a);
      split(a, s[0], t);
      s[0] += t;
      sum(s);
      q = rsqrtf(s[0] * inv + A.eps);
      if (there) {
#pragma unroll
        for (int k = 0; k < H; k++) v[k] = fma2(mul2(v[k], pair(q)), w[k], b[k]);
      }
    }
    if (row < A.S.rows) {
      share.store(out + (long long)row * out_ld, v);
      if (stats != nullptr && thread == 0) reinterpret_cast<float2*>(stats)[row] = there ? make_float2(mean, q) : make_float2(0.f, 0.f);
    }
  }
  copies_but<0>();
}

// dx = q (a - mean a - h mean(a h)) row by row, and with SUMS the sums over the block's rows of g h and g, which stay in the
// registers of the threads that hold their columns: parts[block][2][width].
template <class T, class P, bool VEC, bool SPAN, int VALUES, bool SUMS>
__global__ void __launch_bounds__(VALUES == 16 ? 512 : BLOCK) k_norm_backward(NormArgs A, const T* x, long long x_ld, const P* weight,
                                                                              const float* stats, const T* diff, long long diff_ld, T* grad,
                                                                              long long grad_ld, float* parts) {
  constexpr int H = VALUES / 2;
  extern __shared__ __align__(16) char ring[];
  __shared__ float part[2][2][32];
  const int n = SPAN ? blockDim.x : A.threads, thread = SPAN ? threadIdx.x : threadIdx.x & (n - 1);
  const unsigned rows = SPAN ? 1 : BLOCK / n, sub = SPAN ? 0 : threadIdx.x / n;
  const Share<T, VEC, VALUES> share(thread, n, sub, A.width);
  const unsigned stage = share.bytes(blockDim.x, n), ring_at = (unsigned)__cvta_generic_to_shared(ring);
  RowSum<SPAN, 2> sum = {part, A.group};
  wait_for_stream();
  Ahead ahead = {rows, sub};
  unsigned coming = blockIdx.x;
  auto fetch = [&](int slot, int turn) {
    const bool there = ahead.there();
    if (there) {
      const long long row = coming * rows + sub;
      share.fetch(ring_at + 2 * slot * stage, x + row * x_ld);
      share.fetch(ring_at + (2 * slot + 1) * stage, diff + row * diff_ld);
    }
    copies_end_group();
    ahead.filled |= (unsigned)there << turn;
    coming += gridDim.x;
    ahead.look(A, coming);
  };
  ahead.look(A, coming);
#pragma unroll
  for (int k = 0; k < STAGES<T> - 1; k++) fetch(k, k);
  Pair w[H], dw[H], db[H];
  share.parameters(weight, 1.f, w);
#pragma unroll
  for (int k = 0; k < H; k++) dw[k] = db[k] = pair(0.f);
  const float inv = 1.f / (float)A.width;
  float2 st_next = make_float2(0.f, 0.f);
  if (ahead.filled & 1) st_next = reinterpret_cast<const float2*>(stats)[blockIdx.x * rows + sub];
  int slot = 0;
  for (unsigned tile = blockIdx.x; tile < A.tiles; tile += gridDim.x) {
    if (!VEC && !SPAN) __syncwarp();
    fetch(slot == 0 ? STAGES<T> - 1 : slot - 1, STAGES<T> - 1);
    const float2 st = st_next;
    if (ahead.filled & 2) st_next = reinterpret_cast<const float2*>(stats)[(tile + gridDim.x) * rows + sub];
    copies_but<STAGES<T> - 1>();
    if (!VEC) {
      if (SPAN) __syncthreads();
      else __syncwarp();
    }
    const bool there = ahead.filled & 1;
    ahead.filled >>= 1;
    const unsigned row = tile * rows + sub;
    Pair v[H], g[H];
    if (there) {
      share.take(ring + 2 * slot * stage, x + (long long)row * x_ld, v);
      share.take(ring + (2 * slot + 1) * stage, diff + (long long)row * diff_ld, g);
    } else {
#pragma unroll
      for (int k = 0; k < H; k++) v[k] = g[k] = pair(0.f);
    }
    slot = slot == STAGES<T> - 1 ? 0 : slot + 1;
    if (!SPAN || there) {
      float s[2], t;
      Pair a = pair(0.f), c = pair(0.f);
#pragma unroll
      for (int k = 0; k < H; k++) {
        v[k] = mul2(add2(v[k], pair(there ? -st.x : 0.f)), pair(there ? st.y : 0.f));
        if (SUMS) {
          dw[k] = fma2(g[k], v[k], dw[k]);
          db[k] = add2(db[k], g[k]);
        }
        g[k] = mul2(g[k], w[k]);
        a = add2(a, g[k]);
        c = fma2(g[k], v[k], c);
      }
      split(a, s[0], t);
      s[0] += t;
      split(c, s[1], t);
      s[1] += t;
      sum(s);
      if (there) {
        const float s0 = -s[0] * inv, s1 = -s[1] * inv;
#pragma unroll
        for (int k = 0; k < H; k++) v[k] = mul2(fma2(v[k], pair(s1), add2(g[k], pair(s0))), pair(st.y));
      }
    }
    if (row < A.S.rows) share.store(grad + (long long)row * grad_ld, v);
  }
  copies_but<0>();
  if (!SUMS) return;
  float* mine = parts + (size_t)blockIdx.x * 2 * A.width;
  if (SPAN) {
#pragma unroll
    for (int i = 0; i < VALUES; i += 2) {
      float f0, f1;
      split(dw[i / 2], f0, f1);
      if (share.valid(i)) mine[share.col(i)] = f0;
      if (share.valid(i + 1)) mine[share.col(i + 1)] = f1;
      split(db[i / 2], f0, f1);
      if (share.valid(i)) mine[A.width + share.col(i)] = f0;
      if (share.valid(i + 1)) mine[A.width + share.col(i + 1)] = f1;
    }
  } else {
    // rows of a warp, then the warps
    __shared__ float all[2][BLOCK / 32][VALUES * 32];
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < VALUES; i += 2) {
      float f[4];
      split(dw[i / 2], f[0], f[1]);
      split(db[i / 2], f[2], f[3]);
      for (int o = 16; o >= n; o >>= 1) {
#pragma unroll
        for (int k = 0; k < 4; k++) f[k] += __shfl_xor_sync(0xffffffffu, f[k], o);
      }
      if (lane < n) {
#pragma unroll
        for (int k = 0; k < 4; k++) all[k / 2][threadIdx.x / 32][share.col(i + k % 2)] = f[k];
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
#pragma unroll 8
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
  RowSum<true, 1> sum = {part, WIDE_THREADS / 32};
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
  RowSum<true, 2> sum = {part, WIDE_THREADS / 32};
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
  int values, threads, block, group;  // a thread's values of a row; threads of a row, of a block; see NormArgs
  unsigned tiles, forward, blocks;    // blocks of the two passes; the sums of the backward pass go by its blocks
  unsigned per;                       // rows of a block of the wide sums
  size_t bytes;
};

NormPlan norm_plan(unsigned rows, int width) {
  NormPlan p = {};
  p.wide = width > WIDE;
  if (p.wide) {
    p.blocks = rows / 64 < 1 ? 1 : rows / 64 > 64 ? 64 : rows / 64;
    p.per = (rows + p.blocks - 1) / p.blocks;
  } else {
    p.values = width > MIDDLE ? 16 : 8;
    p.threads = 1;
    while (p.threads < 32 && p.threads * p.values < width) p.threads *= 2;
    if (p.threads * p.values < width) p.threads = (width + p.values * 32 - 1) / (p.values * 32) * 32;
    p.block = p.threads > 32 ? p.threads : BLOCK;
    p.group = p.threads;
    if (p.threads > 32)
      for (p.group = 1; p.group < p.threads / 32;) p.group *= 2;
    const unsigned per = p.threads > 32 ? 1 : BLOCK / p.threads;
    p.tiles = (rows + per - 1) / per;
    // blocks an SM holds: by the stages of float32, whatever the type, so that sums go by the sizes alone, and by registers
    const size_t ring = (size_t)2 * STAGES<float> * p.block * p.values * 4;
    auto fit = [&](size_t smem, int threads) {
      const unsigned by_smem = (unsigned)((224 << 10) / (smem + 1024)), by_threads = threads > p.block ? threads / p.block : 1;
      const unsigned all = 148 * (by_smem < by_threads ? by_smem : by_threads);
      return p.tiles < all ? p.tiles : all;
    };
    p.blocks = fit(ring, p.values == 16 ? 512 : 1024);
    p.forward = fit(ring / 2, p.values == 16 ? 1024 : 1536);
  }
  p.bytes = 256 + (size_t)p.blocks * 2 * width * 4;
  return p;
}

// dynamic shared memory of a pass over `arrays` arrays
template <class T>
size_t ring_bytes(const NormPlan& p, bool vec, int arrays) {
  const unsigned stage = p.values == 16 ? (vec ? Share<T, true, 16>::bytes(p.block, p.threads) : Share<T, false, 16>::bytes(p.block, p.threads))
                                        : (vec ? Share<T, true, 8>::bytes(p.block, p.threads) : Share<T, false, 8>::bytes(p.block, p.threads));
  return (size_t)arrays * STAGES<T> * stage;
}

// F(T, P) for the element types of vectors and parameters, which agree or the latter are float32
template <class F>
cudaError_t by_types(int type, int weight_type, F f) {
  if (type == LMG_FLOAT32) return f(float(), float());
  if (type == LMG_BFLOAT16) return weight_type == LMG_FLOAT32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
  return weight_type == LMG_FLOAT32 ? f(__half(), float()) : f(__half(), __half());
}

template <class T, class P>
auto by_plan(const NormPlan& p, bool vec, bool sums) {
  if (p.values == 16)
    return vec ? (sums ? k_norm_backward<T, P, true, true, 16, true> : k_norm_backward<T, P, true, true, 16, false>)
               : (sums ? k_norm_backward<T, P, false, true, 16, true> : k_norm_backward<T, P, false, true, 16, false>);
  if (p.threads > 32)
    return vec ? (sums ? k_norm_backward<T, P, true, true, 8, true> : k_norm_backward<T, P, true, true, 8, false>)
               : (sums ? k_norm_backward<T, P, false, true, 8, true> : k_norm_backward<T, P, false, true, 8, false>);
  return vec ? (sums ? k_norm_backward<T, P, true, false, 8, true> : k_norm_backward<T, P, true, false, 8, false>)
             : (sums ? k_norm_backward<T, P, false, false, 8, true> : k_norm_backward<T, P, false, false, 8, false>);
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
  NormArgs A = {to_slots(rows, 0), width, 0, 0, 0, eps};
  const NormPlan p = norm_plan(A.S.rows, width);
  A.threads = p.threads;
  A.group = p.group;
  A.tiles = p.tiles;
  const bool vec = rows_aligned(x) && rows_aligned(out);
  const cudaError_t e = by_types(x->type, weight_type, [&](auto t, auto q) {
    typedef decltype(t) T;
    typedef decltype(q) P;
    auto kernel = k_norm_wide<T, P>;
    if (!p.wide && p.values == 16) kernel = vec ? k_norm<T, P, true, true, 16> : k_norm<T, P, false, true, 16>;
    else if (!p.wide && p.threads > 32) kernel = vec ? k_norm<T, P, true, true, 8> : k_norm<T, P, false, true, 8>;
    else if (!p.wide) kernel = vec ? k_norm<T, P, true, false, 8> : k_norm<T, P, false, false, 8>;
    const size_t ring = p.wide ? 0 : ring_bytes<T>(p, vec, 1);
    const cudaError_t e = allow_smem(kernel, ring);
    if (e != cudaSuccess) return e;
    return launch_early(kernel, dim3(p.wide ? A.S.rows : p.forward), p.wide ? WIDE_THREADS : p.block, ring, (cudaStream_t)stream, A,
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
  NormArgs A = {to_slots(rows, 0), width, 0, 0, 0, 0.f};
  const NormPlan p = norm_plan(A.S.rows, width);
  A.threads = p.threads;
  A.group = p.group;
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
      auto kernel = by_plan<T, P>(p, vec, sums);
      const size_t ring = ring_bytes<T>(p, vec, 2);
      if ((e = allow_smem(kernel, ring)) != cudaSuccess) return e;
      e = launch_early(kernel, dim3(p.blocks), p.block, ring, st, A, xp, x->ld, static_cast<const P*>(weight), stats, gp, diff->ld, to,
                       x_gradients->ld, parts);
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

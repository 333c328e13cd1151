// Layer norm over the last dimension and its gradients.
#include "lmg_vectors.h"

namespace lmg {
namespace {

constexpr int BLOCK = 256;      // threads of a block whose rows each lie within a warp
constexpr int WIDE = 8192;      // columns; beyond it rows are read more than once (k_norm_wide, ...)
constexpr int NARROW = 64;      // columns up to which a thread holds eight values of a row, sixteen beyond: 100000 rows of 64 float32 13.5
                                // and 14.0 us (gradients of x), 50000 of 128 bfloat16 10.6 and 8.9
// rows that are in use or on their way; both arrays of the widest rows fit an SM: 3 x 2 x 32 KB of float32, 4 x 2 x 16 KB of 16 bits
template <class T> constexpr int STAGES = sizeof(T) == 4 ? 3 : 4;

__device__ __forceinline__ void copy_async(unsigned to, const void* from, unsigned bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async8(unsigned to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
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

// A thread's VALUES values of the rows it works on: whole pieces of 16 bytes of memory, so that it copies, reads and writes 16
// bytes at a time and waits for no one else's copies.  Rows that do not begin on 16 bytes have their first columns `shift` values
// into the first piece; rows of one thread are as many apart as it takes for all to begin alike.  Copies are asynchronous, into a
// ring in shared memory: rows under way take no registers.
template <class T, int VALUES>
struct Share {
  static constexpr int PER = 16 / sizeof(T), PIECES = VALUES / PER;
  int thread, n, width, shift, before;  // `before`: the values of its first piece that are not the row's yet
  bool full;              // all its values are the row's
  unsigned whole;         // a bit for each piece that is the row's
  unsigned size[PIECES];  // bytes up to the row's end
  unsigned off[PIECES];   // from its first piece, in values

  static __host__ __device__ __forceinline__ unsigned bytes(unsigned block) { return block * PIECES * 16; }  // of a stage
  __device__ __forceinline__ int col(int i) const { return (thread + n * (i / PER)) * PER + i % PER - shift; }
  __device__ __forceinline__ bool valid(int i) const { return i % PER * (int)sizeof(T) < (int)size[i / PER] && (i >= PER || i >= before); }

  __device__ __forceinline__ Share(int thread_, int n_, int shift_, int width_) : thread(thread_), n(n_), width(width_), shift(shift_) {
    before = thread == 0 ? shift : 0;
    whole = 0;
#pragma unroll
    for (int k = 0; k < PIECES; k++) {
      const int left = (width - col(k * PER)) * (int)sizeof(T);
      size[k] = left < 0 ? 0 : left < 16 ? left : 16;
      off[k] = left > 0 ? n * PER * k : 0;
      whole |= (unsigned)(valid(k * PER) && valid(k * PER + PER - 1)) << k;
    }
    full = whole == (1u << PIECES) - 1;
  }
  // where its first piece of a row begins
  template <class Q>
  __device__ __forceinline__ Q* first(Q* row) const { return row - shift + (col(0) < width ? thread * PER : 0); }
  __device__ __forceinline__ void fetch(unsigned stage, const T* at) const {
#pragma unroll
    for (int k = 0; k < PIECES; k++) copy_async(stage + (threadIdx.x + k * blockDim.x) * 16, at + off[k], size[k]);
  }
  __device__ __forceinline__ void take(const char* stage, Pair (&v)[VALUES / 2]) const {
#pragma unroll
    for (int k = 0; k < PIECES; k++) {  // what lies behind the row's end has been filled with zeros
      const uint4 a = *reinterpret_cast<const uint4*>(stage + (threadIdx.x + k * blockDim.x) * 16);
      if constexpr (sizeof(T) == 4) {
        v[2 * k] = pair(__uint_as_float(a.x), __uint_as_float(a.y));
        v[2 * k + 1] = pair(__uint_as_float(a.z), __uint_as_float(a.w));
      } else {
        v[4 * k] = unpack<T>(a.x), v[4 * k + 1] = unpack<T>(a.y), v[4 * k + 2] = unpack<T>(a.z), v[4 * k + 3] = unpack<T>(a.w);
      }
    }
    if (before != 0) {
#pragma unroll
      for (int i = 0; i < PER; i += 2) {
        float f0, f1;
        split(v[i / 2], f0, f1);
        v[i / 2] = pair(i < before ? 0.f : f0, i + 1 < before ? 0.f : f1);
      }
    }
  }
  __device__ __forceinline__ void store(T* at, const Pair (&v)[VALUES / 2]) const {
#pragma unroll
    for (int k = 0; k < PIECES; k++) {
      T* to = at + off[k];
      uint4 a;
      if constexpr (sizeof(T) == 4) {
        float f[4];
        split(v[2 * k], f[0], f[1]);
        split(v[2 * k + 1], f[2], f[3]);
        a = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      } else {
        a = make_uint4(packed<T>(v[4 * k]), packed<T>(v[4 * k + 1]), packed<T>(v[4 * k + 2]), packed<T>(v[4 * k + 3]));
      }
      if (whole >> k & 1) {
        *reinterpret_cast<uint4*>(to) = a;
      } else {
        const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < PER; i++)
          if (valid(k * PER + i)) to[i] = e[i];
      }
    }
  }
  // values that are not the row's to zero
  __device__ __forceinline__ void cut(Pair (&v)[VALUES / 2]) const {
    if (full) return;
#pragma unroll
    for (int k = 0; k < PIECES; k++) {
      if (whole >> k & 1) continue;
#pragma unroll
      for (int i = k * PER; i < k * PER + PER; i += 2) {
        float f0, f1;
        split(v[i / 2], f0, f1);
        v[i / 2] = pair(valid(i) ? f0 : 0.f, valid(i + 1) ? f1 : 0.f);
      }
    }
  }
  template <class P>
  __device__ __forceinline__ void parameters(const P* p, float otherwise, Pair (&w)[VALUES / 2]) const {
#pragma unroll
    for (int i = 0; i < VALUES; i += 2)
      w[i / 2] = pair(p != nullptr && valid(i) ? to_float(p[col(i)]) : otherwise, p != nullptr && valid(i + 1) ? to_float(p[col(i + 1)]) : otherwise);
  }
};

// Sums over the threads of a row, the same for all of them: `n` lanes next to each other, or (SPAN) a block of up to WARPS warps.  A
// block's sums take turns with two places in shared memory, so one barrier a sum is enough.
template <bool SPAN, int SUMS, int WARPS = 16>
struct RowSum {
  float (*part)[SUMS][32];
  int n, turn = 0;
  __device__ __forceinline__ RowSum(float (*part_)[SUMS][32], int n_) : part(part_), n(n_) {
    if (SPAN) {  // the places of warps that the block does not have
      for (int i = threadIdx.x; i < 2 * SUMS * 32; i += blockDim.x) part[i / (SUMS * 32)][i / 32 % SUMS][i % 32] = 0.f;
      __syncthreads();
    }
  }
  template <int FROM>
  static __device__ __forceinline__ void lanes(float (&v)[SUMS]) {
#pragma unroll
    for (int o = FROM / 2; o; o >>= 1) {
#pragma unroll
      for (int s = 0; s < SUMS; s++) v[s] += __shfl_xor_sync(0xffffffffu, v[s], o);
    }
  }
  __device__ __forceinline__ void operator()(float (&v)[SUMS]) {
    if (SPAN) {
      lanes<32>(v);
      const int lane = threadIdx.x & 31;
      float (*p)[32] = part[turn];
      turn ^= 1;
      if (lane == 0) {
#pragma unroll
        for (int s = 0; s < SUMS; s++) p[s][threadIdx.x / 32] = v[s];
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < SUMS; s++) v[s] = p[s][lane & (WARPS - 1)];
      lanes<WARPS>(v);
    } else {
      for (int o = n >> 1; o; o >>= 1) {
#pragma unroll
        for (int s = 0; s < SUMS; s++) v[s] += __shfl_xor_sync(0xffffffffu, v[s], o);
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

// The rows of a block one after the other: which of them hold anything, looked up a turn before their copies begin.
struct Ahead {
  unsigned tile, row, rows;  // whose copies come next
  unsigned filled;           // bit k: the row k turns from now
  int count, place;
  __device__ __forceinline__ void look(const NormArgs& A) {
    place = 0;
    count = tile < A.tiles && row < A.S.rows;
    if (A.S.n_atoms != nullptr && count != 0) {
      const unsigned b = A.S.by_n(row);
      place = (int)(row - b * A.S.n);
      count = A.S.n_atoms[b];
    }
  }
  __device__ __forceinline__ Ahead(const NormArgs& A, unsigned rows_, unsigned sub)
      : tile(blockIdx.x), row(blockIdx.x * rows_ + sub), rows(rows_ * gridDim.x), filled(0) {
    look(A);
  }
  // whether the next row's copies are to begin
  __device__ __forceinline__ bool next(const NormArgs& A, int turn) {
    const bool there = place < count;
    filled |= (unsigned)there << turn;
    tile += gridDim.x;
    row += rows;
    look(A);
    return there;
  }
};

// how many values before it the 16 bytes begin that a row begins in
template <class T>
__device__ __forceinline__ int shift_of(const T* row) { return (int)(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T); }

// Layer norm with the row in registers: mean, then the squares of what is left.  A block goes from row to row with its weights in
// registers.  16384 rows of 4096 bfloat16: 104 us with the next row in registers; 91 us with the ring, bound by what it issued with eight
// values a thread, one at a time and each checked against the row's end; 67 us with sixteen in pairs, 54 with registers for one wave of
// blocks, 50 with the row's edges seen to only where they are.
template <class T, class P, bool SPAN, int VALUES>
__global__ void __maxnreg__(VALUES == 16 ? 80 : 64) k_norm(NormArgs A, const T* x, long long x_ld, const P* weight, const P* bias, T* out,
                                                             long long out_ld, float* stats) {
  constexpr int H = VALUES / 2, S = STAGES<T>;
  extern __shared__ __align__(16) char ring[];
  __shared__ float part[2][1][32];
  const int n = SPAN ? blockDim.x : A.threads, thread = SPAN ? threadIdx.x : threadIdx.x & (n - 1);
  const unsigned rows = SPAN ? 1 : BLOCK / n, sub = SPAN ? 0 : threadIdx.x / n;
  unsigned row = blockIdx.x * rows + sub;
  const Share<T, VALUES> share(thread, n, shift_of(x + (long long)row * x_ld), A.width);
  const unsigned stage = share.bytes(blockDim.x), ring_at = (unsigned)__cvta_generic_to_shared(ring);
  RowSum<SPAN, 1> sum(part, n);
  wait_for_stream();
  const T* from = share.first(x + (long long)row * x_ld);
  T* to = share.first(out + (long long)row * out_ld);
  const long long x_jump = x_ld * rows * gridDim.x, out_jump = out_ld * rows * gridDim.x;
  Ahead ahead(A, rows, sub);
#pragma unroll
  for (int k = 0; k < S - 1; k++) {
    if (ahead.next(A, k)) share.fetch(ring_at + k * stage, from);
    copies_end_group();
    from += x_jump;
  }
  Pair w[H], b[H];
  share.parameters(weight, 1.f, w);
  share.parameters(bias, 0.f, b);
  const float inv = 1.f / (float)A.width;
  unsigned at = 0, fill = (S - 1) * stage;  // the stage in use, and the one before it, which is filled next
  for (unsigned tile = blockIdx.x; tile < A.tiles; tile += gridDim.x) {
    if (ahead.next(A, S - 1)) share.fetch(ring_at + fill, from);
    copies_end_group();
    from += x_jump;
    copies_but<S - 1>();
    const bool there = ahead.filled & 1;
    ahead.filled >>= 1;
    Pair v[H];
    if (there) {
      share.take(ring + at, v);
    } else {
#pragma unroll
      for (int k = 0; k < H; k++) v[k] = pair(0.f);
    }
    fill = at;
    at = at == (S - 1) * stage ? 0 : at + stage;
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
      const Pair minus = pair(-mean);
#pragma unroll
      for (int k = 0; k < H; k++) v[k] = add2(v[k], minus);
      share.cut(v);
      a = mul2(v[0], v[0]);
#pragma unroll
      for (int k = 1; k < H; k++) a = fma2(v[k], v[k], a);
      split(a, s[0], t);
      s[0] += t;
      sum(s);
      q = rsqrtf(s[0] * inv + A.eps);
      if (there) {
        const Pair qq = pair(q);
#pragma unroll
        for (int k = 0; k < H; k++) v[k] = fma2(mul2(v[k], qq), w[k], b[k]);
      }
    }
    if (SPAN || row < A.S.rows) {
      share.store(to, v);
      if (stats != nullptr && thread == 0) reinterpret_cast<float2*>(stats)[row] = there ? make_float2(mean, q) : make_float2(0.f, 0.f);
    }
    row += rows * gridDim.x;
    to += out_jump;
  }
  copies_but<0>();
}

// dx = q (a - mean a - h mean(a h)) row by row, and with SUMS the sums over the block's rows of g h and g, which stay in the
// registers of the threads that hold their columns: parts[block][2][width].
template <class T, class P, bool SPAN, int VALUES, bool SUMS>
__global__ void __maxnreg__(VALUES == 16 ? 128 : 80) k_norm_backward(NormArgs A, const T* x, long long x_ld, const P* weight, const float* stats,
                                                                      const T* diff, long long diff_ld, T* grad, long long grad_ld, float* parts, P* dweight, P* dbias) {
  constexpr int H = VALUES / 2, S = STAGES<T>;
  extern __shared__ __align__(16) char ring[];
  __shared__ float part[2][2][32];
  const int n = SPAN ? blockDim.x : A.threads, thread = SPAN ? threadIdx.x : threadIdx.x & (n - 1);
  const unsigned rows = SPAN ? 1 : BLOCK / n, sub = SPAN ? 0 : threadIdx.x / n;
  unsigned row = blockIdx.x * rows + sub;
  const Share<T, VALUES> share(thread, n, shift_of(x + (long long)row * x_ld), A.width);
  // a stage holds both arrays and, for every thread, its row's stats: one row ahead in registers they were waited for at each turn's end
  // (16384 rows of 4096 bfloat16: 107 us instead of 76)
  const unsigned array = share.bytes(blockDim.x), stage = 2 * array + blockDim.x * 8, ring_at = (unsigned)__cvta_generic_to_shared(ring);
  RowSum<SPAN, 2> sum(part, n);
  wait_for_stream();
  if (SUMS && gridDim.x > 1) no_status(parts);
  const T *x_from = share.first(x + (long long)row * x_ld), *g_from = share.first(diff + (long long)row * diff_ld);
  T* to = share.first(grad + (long long)row * grad_ld);
  const unsigned jump = rows * gridDim.x;
  const long long x_jump = x_ld * jump, g_jump = diff_ld * jump, to_jump = grad_ld * jump;
  const float* st_from = stats + 2ll * row;
  Ahead ahead(A, rows, sub);
  auto fetch = [&](unsigned fill, int turn) {
    if (ahead.next(A, turn)) {
      share.fetch(ring_at + fill, x_from);
      share.fetch(ring_at + fill + array, g_from);
      copy_async8(ring_at + fill + 2 * array + threadIdx.x * 8, st_from);
    }
    copies_end_group();
    x_from += x_jump;
    g_from += g_jump;
    st_from += 2 * jump;
  };
#pragma unroll
  for (int k = 0; k < S - 1; k++) fetch(k * stage, k);
  Pair w[H], dw[H], db[H];
  share.parameters(weight, 1.f, w);
#pragma unroll
  for (int k = 0; k < H; k++) dw[k] = db[k] = pair(0.f);
  const float inv = 1.f / (float)A.width;
  unsigned at = 0, fill = (S - 1) * stage;
  for (unsigned tile = blockIdx.x; tile < A.tiles; tile += gridDim.x) {
    fetch(fill, S - 1);
    copies_but<S - 1>();
    const bool there = ahead.filled & 1;
    ahead.filled >>= 1;
    Pair v[H], g[H];
    float2 st = make_float2(0.f, 0.f);
    if (there) {
      share.take(ring + at, v);
      share.take(ring + at + array, g);
      st = *reinterpret_cast<const float2*>(ring + at + 2 * array + threadIdx.x * 8);
    } else {
#pragma unroll
      for (int k = 0; k < H; k++) v[k] = g[k] = pair(0.f);
    }
    fill = at;
    at = at == (S - 1) * stage ? 0 : at + stage;
    if (!SPAN || there) {
      float s[2], t;
      Pair a = pair(0.f), c = pair(0.f);
      const Pair minus = pair(-st.x), q = pair(st.y);
#pragma unroll
      for (int k = 0; k < H; k++) {
        v[k] = mul2(add2(v[k], minus), q);
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
        const Pair s0 = pair(-s[0] * inv), s1 = pair(-s[1] * inv);
#pragma unroll
        for (int k = 0; k < H; k++) v[k] = mul2(fma2(v[k], s1, add2(g[k], s0)), q);
      }
    }
    if (SPAN || row < A.S.rows) share.store(to, v);
    row += jump;
    to += to_jump;
  }
  copies_but<0>();
  if (!SUMS) return;
  // The block's sums by way of the ring, so that neighbouring threads write neighbouring columns (each thread its own columns: 690 rows of 5984
  // bfloat16 22.8 us instead of 16.8); or the call's, where one block does all.
  float* all = reinterpret_cast<float*>(ring);
  // a column's place: a word more every 32, or rows of an odd pitch, for which no division is needed; rows that no thread has had are left out
  const int used = min((int)rows, (int)A.S.rows), pitch = A.width | 1;
  auto place = [&](int which, int r, int c) -> float& {
    const int at = SPAN ? which * A.width + c : (which * used + r) * pitch + c;
    return all[SPAN ? at + at / 32 : at];
  };
  auto put = [&](int which, int c, float v) {
    if (gridDim.x > 1) {
      parts[((size_t)blockIdx.x * 2 + which) * A.width + c] = v;
    } else {
      P* to = which ? dbias : dweight;
      if (to != nullptr) to[c] = from_float<P>(v);
    }
  };
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VALUES; i += 2) {
    float f[4];
    split(dw[i / 2], f[0], f[1]);
    split(db[i / 2], f[2], f[3]);
#pragma unroll
    for (int k = 0; k < 4; k++)
      if ((SPAN || (int)sub < used) && share.valid(i + k % 2)) place(k / 2, sub, share.col(i + k % 2)) = f[k];
  }
  __syncthreads();
  if (SPAN) {
    for (int c = threadIdx.x; c < 2 * A.width; c += blockDim.x) put(c >= A.width, c >= A.width ? c - A.width : c, all[c + c / 32]);
  } else {
    // columns by as many threads as there are, a power of two of them a column, which take rows in turn
    int together = 1;
    while (together < 32 && A.width * together * 2 <= BLOCK) together *= 2;
    const int part_of = threadIdx.x & (together - 1);
    for (int c0 = 0; c0 < 2 * A.width; c0 += BLOCK / together) {
      const int c = c0 + threadIdx.x / together, which = c >= A.width;
      float t = 0.f;
      if (c < 2 * A.width) {
#pragma unroll 8
        for (int r = part_of; r < used; r += together) t += place(which, r, c - which * A.width);
      }
      for (int o = together >> 1; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      if (c < 2 * A.width && part_of == 0) put(which, c - which * A.width, t);
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

// ---- rows of more than WIDE columns, and of any width where the arrays begin differently in their 16 bytes: a block a row, read again for each
// sum (from the L1, which holds a row of 200 KB).  2000 rows of 16384 bfloat16 57 us and 130 for the gradients, 0.35 and 0.23 of the measured bandwidth.
// Narrow rows are what it serves badly: 200000 of 28 float32, 29 apart, to dense ones 1384 and 1190 us (10.7 and 18.9 where both lie alike).
constexpr int WIDE_THREADS = 1024;

template <class T, class P>
__global__ void __launch_bounds__(WIDE_THREADS) k_norm_wide(NormArgs A, const T* x, long long x_ld, const P* weight, const P* bias, T* out,
                                                            long long out_ld, float* stats) {
  __shared__ float part[2][1][32];
  RowSum<true, 1, WIDE_THREADS / 32> sum(part, 0);
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
  RowSum<true, 2, WIDE_THREADS / 32> sum(part, 0);
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
  no_status(parts);
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
// Which kernels: by the sizes, and by `slack`, the values that the rows' first pieces of 16 bytes may have more than the rows.
struct NormPlan {
  bool wide;
  int values, threads, block;       // a thread's values of a row; threads of a row, of a block
  unsigned rows;                    // that a block has at once
  unsigned tiles, forward, blocks;  // blocks of the two passes
  unsigned per;                     // rows of a block of the wide sums
  size_t bytes;
};

NormPlan norm_plan(unsigned rows, int width, int slack) {
  NormPlan p = {};
  p.wide = width + slack > WIDE;
  if (p.wide) {
    p.blocks = rows / 64 < 1 ? 1 : rows / 64 > 64 ? 64 : rows / 64;
    p.per = (rows + p.blocks - 1) / p.blocks;
  } else {
    const int most = width + slack;
    p.values = most > NARROW ? 16 : 8;
    p.threads = 1;
    while (p.threads < 32 && p.threads * p.values < most) p.threads *= 2;
    if (p.threads * p.values < most) p.threads = (most + p.values * 32 - 1) / (p.values * 32) * 32;
    p.block = p.threads > 32 ? p.threads : BLOCK;
    const unsigned per = p.threads > 32 ? 1 : BLOCK / p.threads;
    p.rows = per;
    p.tiles = (rows + per - 1) / per;
    // blocks an SM holds: by the stages of float32, whatever the type, so that sums go by the sizes alone, and by registers.  148 and its
    // multiples by a block's rows, or by 2: as many rows apart as it takes for a thread's rows to begin alike in their 16 bytes
    const size_t ring = (size_t)STAGES<float> * p.block * (2 * p.values * 4 + 8);
    auto fit = [&](size_t smem, int threads) {
      const unsigned by_smem = (unsigned)((224 << 10) / (smem + 1024)), by_threads = threads > p.block ? threads / p.block : 1;
      unsigned all = 148 * (by_smem < by_threads ? by_smem : by_threads);
      if (per == 1 && slack) all = all / 8 * 8;
      return p.tiles < all ? p.tiles : all;
    };
    p.blocks = fit(ring, p.values == 16 ? 512 : 768);
    p.forward = fit(ring / 2, p.values == 16 ? 768 : 1024);
    // four rows a block and more, so that the sums are no more than the rows; one block needs no other launch for them (2.8 us)
    if (per == 1 && p.blocks > 148 && p.blocks > p.tiles / 4) p.blocks = p.tiles / 4 > 148 ? p.tiles / 4 / 8 * 8 : 148;
    if (p.blocks > p.tiles) p.blocks = p.tiles;
    const bool any = per > 1 || slack == 0;  // number of blocks lets a thread's rows begin alike
    if (!any && p.blocks < p.tiles) p.blocks = p.blocks / 8 * 8;
    if (any && p.tiles <= 4) p.blocks = 1;
  }
  p.bytes = STATUS_FRONT + (size_t)p.blocks * 2 * width * 4;
  return p;
}

// Rows that begin alike in their 16 bytes wherever one thread meets them: those of one array and, for one row, of all arrays.  false: they are
// the wide kernels'.
bool alike(const lmg_vectors* a, const lmg_vectors* b) {
  const size_t size = element_bytes(a->type);
  return (reinterpret_cast<uintptr_t>(a->data) - reinterpret_cast<uintptr_t>(b->data)) % 16 == 0 && (size_t)(a->ld - b->ld) * size % 16 == 0;
}

NormPlan plan_of(unsigned rows, int width, const lmg_vectors* x, bool all_alike) {
  if (!all_alike) return norm_plan(rows, width, WIDE);
  return norm_plan(rows, width, rows_aligned(x) ? 0 : 16 / (int)element_bytes(x->type) - 1);
}

// Threads keep the place in 16 bytes at which their first row begins: a pass whose threads have more than one has to jump by whole ones.
int check_jump(const NormPlan& p, unsigned blocks, const lmg_vectors* x) {
  if (p.wide || blocks >= p.tiles || (unsigned long long)p.rows * blocks * x->ld * element_bytes(x->type) % 16 == 0) return LMG_OK;
  return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "rows of a thread begin at different places in their 16 bytes");
}

// dynamic shared memory of a pass over `arrays` arrays
template <class T>
size_t ring_bytes(const NormPlan& p, int arrays) {
  return (size_t)STAGES<T> * (arrays * (p.values == 16 ? Share<T, 16>::bytes(p.block) : Share<T, 8>::bytes(p.block)) + (arrays == 2 ? p.block * 8 : 0));
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
  if (op == LMG_OP_EMBED_BACKWARD) return lmg::embed_backward_bytes((unsigned)rows, ntypes, width);
  size_t most = lmg::norm_plan((unsigned)rows, width, lmg::WIDE).bytes;  // that of any alignment
  for (int slack : {0, 3, 7}) {
    const size_t bytes = lmg::norm_plan((unsigned)rows, width, slack).bytes;
    if (bytes > most) most = bytes;
  }
  return most;
}

void lmg_norm_plan(int rows, int width, int slack, unsigned plan[5]) {
  const lmg::NormPlan p = lmg::norm_plan((unsigned)rows, width, slack);
  plan[0] = p.wide;
  plan[1] = p.rows;
  plan[2] = p.tiles;
  plan[3] = p.forward;
  plan[4] = p.blocks;
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
  const NormPlan p = plan_of(A.S.rows, width, x, alike(x, out));
  if ((rc = check_jump(p, p.forward, x))) return rc;
  A.threads = p.threads;
  A.tiles = p.tiles;
  const cudaError_t e = by_types(x->type, weight_type, [&](auto t, auto q) {
    typedef decltype(t) T;
    typedef decltype(q) P;
    auto kernel = k_norm_wide<T, P>;
    if (!p.wide && p.threads > 32) kernel = k_norm<T, P, true, 16>;
    else if (!p.wide) kernel = p.values == 16 ? k_norm<T, P, false, 16> : k_norm<T, P, false, 8>;
    const size_t ring = p.wide ? 0 : ring_bytes<T>(p, 1);
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
  NormArgs A = {to_slots(rows, 0), width, 0, 0, 0.f};
  const NormPlan p = none ? norm_plan(0, width, 0) : plan_of(A.S.rows, width, x, alike(x, diff) && alike(x, x_gradients));
  if (!none && (rc = check_jump(p, p.blocks, x))) return rc;
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
  const bool sums = weight_gradients || bias_gradients;
  float* parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + STATUS_FRONT);
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
      auto kernel = sums ? k_norm_backward<T, P, true, 16, true> : k_norm_backward<T, P, true, 16, false>;
      if (p.threads <= 32 && p.values == 16) kernel = sums ? k_norm_backward<T, P, false, 16, true> : k_norm_backward<T, P, false, 16, false>;
      else if (p.threads <= 32) kernel = sums ? k_norm_backward<T, P, false, 8, true> : k_norm_backward<T, P, false, 8, false>;
      const size_t ring = ring_bytes<T>(p, 2);
      if ((e = allow_smem(kernel, ring)) != cudaSuccess) return e;
      e = launch_early(kernel, dim3(p.blocks), p.block, ring, st, A, xp, x->ld, static_cast<const P*>(weight), stats, gp, diff->ld, to,
                       x_gradients->ld, parts, static_cast<P*>(weight_gradients), static_cast<P*>(bias_gradients));
    }
    if (e != cudaSuccess) return e;
    launches++;
    if (!sums || (!p.wide && p.blocks == 1)) return e;
    launches++;
    return launch_early(k_norm_sums<P>, dim3((width + 31) / 32, 2), 1024, 0, st, parts, (int)p.blocks, width, static_cast<P*>(weight_gradients),
                        static_cast<P*>(bias_gradients));
  });
  lmg_internal_count_launches(launches);
  return e == cudaSuccess ? LMG_OK : vectors_cuda(e, "gradients of a layer norm");
}

}  // extern "C"

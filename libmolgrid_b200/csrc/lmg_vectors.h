// What the kernels on learned type vectors share: element types, slots, random bits, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/lmg_b200.h"
#include "lmg_launch.h"

extern "C" void lmg_internal_set_error(const char* msg);
extern "C" void lmg_internal_count_launches(long n);

namespace lmg {

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994)
struct FastDiv {
  unsigned d, mul, shift;
  FastDiv() = default;
  explicit FastDiv(unsigned by) : d(by), shift(by > 1 ? 32 - __builtin_clz(by - 1) : 0) {
    mul = (unsigned)(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ unsigned operator()(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
#endif
};

constexpr size_t STATUS_FRONT = 256;  // bytes of a workspace before the scratch of these calls

struct Slots {
  unsigned rows, n;  // batch * max_atoms, max_atoms
  FastDiv by_n;
  const int* n_atoms;
  const void* index;
  int index_type;
  int ntypes;
  int* status;
};

struct Drop {
  unsigned upper, lower;  // p * 2^32 = upper * 65536 + lower; 2^32 itself as 65535 and 65536
  float scale;            // 1 / (1 - p)
  unsigned long long seed, offset;
  const unsigned long long* state;
};

#ifdef __CUDACC__
__device__ __forceinline__ bool slot_filled(const Slots& S, unsigned row) {
  if (S.n_atoms == nullptr) return true;
  const unsigned b = S.by_n(row);
  return (int)(row - b * S.n) < S.n_atoms[b];
}

// types of N slots, -1 where one is empty (or `in` is false); all their counts and indices are on their way together
template <int N>
__device__ __forceinline__ void slot_types(const Slots& S, const unsigned (&row)[N], const bool (&in)[N], int (&t)[N]) {
  if (S.index_type == LMG_INDEX_FLOAT32) {
    float f[N];
#pragma unroll
    for (int k = 0; k < N; k++) f[k] = in[k] ? static_cast<const float*>(S.index)[row[k]] : -1.f;
#pragma unroll
    for (int k = 0; k < N; k++) {
      f[k] = roundf(f[k]);
      t[k] = f[k] >= 0.f ? f[k] < 2147483648.f ? (int)f[k] : 0x7fffffff : -1;
    }
  } else if (S.index_type == LMG_INDEX_INT32) {
#pragma unroll
    for (int k = 0; k < N; k++) t[k] = in[k] ? static_cast<const int*>(S.index)[row[k]] : -1;
  } else {
    long long l[N];
#pragma unroll
    for (int k = 0; k < N; k++) l[k] = in[k] ? static_cast<const long long*>(S.index)[row[k]] : -1;
#pragma unroll
    for (int k = 0; k < N; k++) t[k] = l[k] < 0 ? -1 : l[k] < 0x7fffffff ? (int)l[k] : 0x7fffffff;
  }
  if (S.n_atoms != nullptr) {
    int place[N], count[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
      const unsigned b = S.by_n(in[k] ? row[k] : 0);
      place[k] = (int)((in[k] ? row[k] : 0) - b * S.n);
      count[k] = S.n_atoms[b];
    }
#pragma unroll
    for (int k = 0; k < N; k++)
      if (place[k] >= count[k]) t[k] = -1;
  }
  bool high = false;
#pragma unroll
  for (int k = 0; k < N; k++)
    if (t[k] >= S.ntypes) {
      high = true;
      t[k] = -1;
    }
  if (high && S.status != nullptr) *S.status = 1;
}
__device__ __forceinline__ int slot_type(const Slots& S, unsigned row) {
  const unsigned rows[1] = {row};
  const bool in[1] = {true};
  int t[1];
  slot_types(S, rows, in, t);
  return t[0] < 0 ? -1 : t[0];
}

// The front of a workspace is what lmg_check_status() reads: it goes with flags behind it, so the first launch of a call that writes there takes
// it away.
__device__ __forceinline__ void no_status(void* scratch) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *reinterpret_cast<unsigned long long*>(static_cast<char*>(scratch) - STATUS_FRONT) = 0;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <int N> struct Bytes;
template <> struct Bytes<16> { typedef uint4 type; };
template <> struct Bytes<8> { typedef uint2 type; };

// COLS values to a row from column `col` on, a multiple of COLS, those behind its end left out; VEC: the row begins on 16 bytes, and they are
// written 16 bytes at a time, or as many as they are
template <class T, int COLS, bool VEC = true>
__device__ __forceinline__ void store_cols(T* row, int col, int width, const float (&v)[COLS]) {
  constexpr int N = !VEC ? COLS : COLS * sizeof(T) < 16 ? COLS : 16 / sizeof(T);
#pragma unroll
  for (int k = 0; k < COLS; k += N) {
    if (VEC && col + k + N <= width) {
      typename Bytes<VEC ? N * sizeof(T) : 16>::type a;
      T* e = reinterpret_cast<T*>(&a);
#pragma unroll
      for (int i = 0; i < N; i++) e[i] = from_float<T>(v[k + i]);
      *reinterpret_cast<typename Bytes<VEC ? N * sizeof(T) : 16>::type*>(row + col + k) = a;
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (col + k + i < width) row[col + k + i] = from_float<T>(v[k + i]);
    }
  }
}

// COLS values of a row as they lie, likewise, zeros behind its end: read long before they are used, in half the registers for 16 bits
template <class T, int COLS, bool VEC = true>
struct Raw {
  static constexpr int WORDS = COLS * sizeof(T) / 4;
  unsigned w[WORDS];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < WORDS; i++) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* row, int col, int width) {
    constexpr int N = !VEC ? COLS : WORDS < 4 ? COLS : 16 / (int)sizeof(T);
#pragma unroll
    for (int k = 0; k < COLS; k += N) {
      unsigned* to = w + k * sizeof(T) / 4;
      if (VEC && col + k + N <= width) {
        if constexpr (N * sizeof(T) == 16) {
          const uint4 a = *reinterpret_cast<const uint4*>(row + col + k);
          to[0] = a.x, to[1] = a.y, to[2] = a.z, to[3] = a.w;
        } else {
          const uint2 a = *reinterpret_cast<const uint2*>(row + col + k);
          to[0] = a.x, to[1] = a.y;
        }
      } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i++) to[i] = col + k + i < width ? __float_as_uint(row[col + k + i]) : 0u;
      } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
        for (int i = 0; i < N; i += 2)
          to[i / 2] = (col + k + i < width ? h[col + k + i] : 0u) | (col + k + i + 1 < width ? (unsigned)h[col + k + i + 1] << 16 : 0u);
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    const unsigned short h = (unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2]);
    return to_float(*reinterpret_cast<const T*>(&h));
  }
};

// Philox4x32-10: ten rounds of two 32 x 32 -> 64 bit products (Salmon, Moraes, Dror and Shaw, 2011, section 4.3), N blocks side by
// side under one key
template <int N>
__device__ __forceinline__ void philox(uint4 (&c)[N], unsigned k0, unsigned k1) {
#pragma unroll
  for (int i = 0; i < 10; i++) {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const unsigned long long a = (unsigned long long)c[j].x * 0xD2511F53u, b = (unsigned long long)c[j].z * 0xCD9E8D57u;
      c[j] = make_uint4((unsigned)(b >> 32) ^ c[j].y ^ k0, (unsigned)b, (unsigned)(a >> 32) ^ c[j].w ^ k1, (unsigned)a);
    }
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// key and offset of a call, read once a thread
struct DropKey {
  unsigned k0, k1, o0, o1;
  __device__ __forceinline__ explicit DropKey(const Drop& D) {
    const unsigned long long s = D.state ? D.state[0] : D.seed, o = D.state ? D.state[1] : D.offset;
    k0 = (unsigned)s;
    k1 = (unsigned)(s >> 32);
    o0 = (unsigned)o;
    o1 = (unsigned)(o >> 32) & 0x7fffffffu;
  }
};

// A block's 128 bits decide eight columns, a half word each, but for a tie with the threshold's upper half (one block in 8192), for
// which as many bits are drawn again: a bit for each column that loses its tie.  Apart, so that what calls it keeps its registers.
static __device__ __noinline__ unsigned lost_ties(uint4 w, unsigned upper, unsigned lower, uint4 counter, unsigned k0, unsigned k1) {
  uint4 v[1] = {make_uint4(counter.x, counter.y, counter.z, counter.w | 0x80000000u)};
  philox(v, k0, k1);
  const unsigned word[4] = {w.x, w.y, w.z, w.w}, low[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
  unsigned lost = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int shift = j & 1 ? 16 : 0;
    if ((word[j / 2] >> shift & 0xffffu) == upper && (low[j / 2] >> shift & 0xffffu) < lower) lost |= 1u << j;
  }
  return lost;
}

// Which columns of a group stay.  Half words are compared where they are: the upper one of a word as the word, the lower one shifted up.
struct Bits8 {
  uint4 w;
  unsigned least, lost;
  __device__ __forceinline__ void set(uint4 words, const Drop& D, const DropKey& K, unsigned row, unsigned group) {
    w = words;
    least = D.upper << 16;
    lost = 0;
    if (D.lower != 0) {
      const unsigned both = least | D.upper;
      // the top bit of a half word is set if it, or one below it, equals the threshold
      const unsigned x = w.x ^ both, y = w.y ^ both, z = w.z ^ both, u = w.w ^ both;
      if ((((x - 0x00010001u) & ~x) | ((y - 0x00010001u) & ~y) | ((z - 0x00010001u) & ~z) | ((u - 0x00010001u) & ~u)) & 0x80008000u)
        lost = lost_ties(w, D.upper, D.lower, make_uint4(group, row, K.o0, K.o1), K.k0, K.k1);
    }
  }
  __device__ __forceinline__ bool reaches(int j) const {
    const unsigned v = j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w;
    return (j & 1 ? v : v << 16) >= least;
  }
  __device__ __forceinline__ unsigned mask() const {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m |= (unsigned)reaches(j) << j;
    return m & ~lost;
  }
  __device__ __forceinline__ void apply(float scale, float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = reaches(j) ? v[j] * scale : 0.f;
    if (lost != 0) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (lost >> j & 1) v[j] = 0.f;
    }
  }
};

// the bits of one group of eight columns
__device__ __forceinline__ unsigned kept8(const Drop& D, const DropKey& K, unsigned row, unsigned group) {
  uint4 c[1] = {make_uint4(group, row, K.o0, K.o1)};
  philox(c, K.k0, K.k1);
  Bits8 b;
  b.set(c[0], D, K, row, group);
  return b.mask();
}
#endif

// ---- host side of the entry points (lmg_embed.cu) -------------------------------------------------------------------
int vectors_fail(int code, const char* msg);
int vectors_cuda(cudaError_t e, const char* what);
// LMG_OK, or the refusal of sizes, an array or a dropout that no call takes
int check_slots(const lmg_slots* s, int width);
int check_vectors(const lmg_vectors* v, int width, const char* name);
int check_drop(const lmg_dropout_spec* d);
int check_index(const lmg_slots* s, int ntypes);
Slots to_slots(const lmg_slots* s, int ntypes);
Drop to_drop(const lmg_dropout_spec* d);  // upper and lower 0: nothing is dropped
inline bool drops(const Drop& D) { return D.upper != 0 || D.lower != 0; }
size_t embed_backward_bytes(unsigned rows, int ntypes, int width);
// f(T, O) for the element types of source and result, which agree or are float32 and 16 bits: NARROW, a float32 source of 16-bit results;
// WIDEN, the other way round
template <bool NARROW, bool WIDEN, class F>
cudaError_t by_vector_types(int in, int out, F f) {
  if constexpr (NARROW) {
    if (in == LMG_FLOAT32 && out == LMG_BFLOAT16) return f(float(), __nv_bfloat16());
    if (in == LMG_FLOAT32 && out == LMG_FLOAT16) return f(float(), __half());
  }
  if constexpr (WIDEN) {
    if (in == LMG_BFLOAT16 && out == LMG_FLOAT32) return f(__nv_bfloat16(), float());
    if (in == LMG_FLOAT16 && out == LMG_FLOAT32) return f(__half(), float());
  }
  if (in == LMG_FLOAT32) return f(float(), float());
  if (in == LMG_BFLOAT16) return f(__nv_bfloat16(), __nv_bfloat16());
  return f(__half(), __half());
}
inline size_t element_bytes(int type) { return type == LMG_FLOAT32 ? 4 : 2; }
// Leave to have more shared memory than the 48 KB of any launch, its own variables among them (17 KB at most here): always for as much as
// any launch wants, so that calls of several threads do not undo one another's, and once for each kernel and device, as far as
// a thread remembers.
constexpr size_t SMEM_MOST = 224 << 10;
cudaError_t allow_smem_of(const void* kernel);
template <class... P>
cudaError_t allow_smem(void (*kernel)(P...), size_t bytes) {
  return bytes <= 31 << 10 ? cudaSuccess : allow_smem_of(reinterpret_cast<const void*>(kernel));
}

// launch_early() of blocks in clusters
template <class... P, class... Q>
inline cudaError_t launch_clusters(void (*kernel)(P...), unsigned blocks, unsigned cluster, unsigned threads, size_t smem, cudaStream_t st, Q... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(blocks);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  c.attrs = attr;
  c.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&c, kernel, args...);
  if (e != cudaSuccess) cudaGetLastError();  // it is in `e`: not to be found again by a later launch
  return e;
}

// rows of which any eight columns that begin at a multiple of eight lie on 16 bytes
inline bool rows_aligned(const lmg_vectors* v) {
  return reinterpret_cast<uintptr_t>(v->data) % 16 == 0 && v->ld * element_bytes(v->type) % 16 == 0;
}
inline size_t aligned256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace lmg

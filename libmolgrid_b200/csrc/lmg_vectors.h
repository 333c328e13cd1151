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
  explicit FastDiv(unsigned by) : d(by), shift(0) {
    while (shift < 32 && (1ull << shift) < by) shift++;
    mul = (unsigned)(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ unsigned operator()(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
#endif
};

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
  unsigned threshold_hi, threshold_lo;  // upper half (up to 65536) and lower half of p * 2^32
  float scale;                          // 1 / (1 - p)
  unsigned long long seed, offset;
  const unsigned long long* state;
};

#ifdef __CUDACC__
__device__ __forceinline__ bool slot_filled(const Slots& S, unsigned row) {
  if (S.n_atoms == nullptr) return true;
  const unsigned b = S.by_n(row);
  return (int)(row - b * S.n) < S.n_atoms[b];
}

// type of a slot, -1 where it is empty
__device__ __forceinline__ int slot_type(const Slots& S, unsigned row) {
  if (!slot_filled(S, row)) return -1;
  bool high;
  int t;
  if (S.index_type == LMG_INDEX_FLOAT32) {
    const float f = roundf(static_cast<const float*>(S.index)[row]);
    if (!(f >= 0.f)) return -1;
    t = f < 2147483648.f ? (int)f : 0x7fffffff;
    high = t >= S.ntypes;
  } else if (S.index_type == LMG_INDEX_INT32) {
    t = static_cast<const int*>(S.index)[row];
    high = t >= S.ntypes;
  } else {
    const long long l = static_cast<const long long*>(S.index)[row];
    high = l >= S.ntypes;
    t = l < 0 ? -1 : (int)l;
  }
  if (high) {
    if (S.status != nullptr) *S.status = 1;
    return -1;
  }
  return t < 0 ? -1 : t;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// eight values of a row from column `col` on, zeros behind its end; VEC: column 0 lies on 16 bytes and `col` is a multiple of 8
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int col, int width, float (&v)[8]) {
  constexpr int N = VEC ? 16 / sizeof(T) : 8;
#pragma unroll
  for (int k = 0; k < 8; k += N) {
    if (VEC && col + k + N <= width) {
      const uint4 a = *reinterpret_cast<const uint4*>(row + col + k);
      const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
      for (int i = 0; i < N; i++) v[k + i] = to_float(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) v[k + i] = col + k + i < width ? to_float(row[col + k + i]) : 0.f;
    }
  }
}

template <class T, bool VEC>
__device__ __forceinline__ void store8(T* row, int col, int width, const float (&v)[8]) {
  constexpr int N = VEC ? 16 / sizeof(T) : 8;
#pragma unroll
  for (int k = 0; k < 8; k += N) {
    if (VEC && col + k + N <= width) {
      uint4 a;
      T* e = reinterpret_cast<T*>(&a);
#pragma unroll
      for (int i = 0; i < N; i++) e[i] = from_float<T>(v[k + i]);
      *reinterpret_cast<uint4*>(row + col + k) = a;
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (col + k + i < width) row[col + k + i] = from_float<T>(v[k + i]);
    }
  }
}

// Philox4x32-10: ten rounds of two 32 x 32 -> 64 bit products (Salmon, Moraes, Dror and Shaw, 2011, section 4.3)
__device__ __forceinline__ uint4 philox(uint4 c, unsigned k0, unsigned k1) {
#pragma unroll
  for (int i = 0; i < 10; i++) {
    const unsigned long long a = (unsigned long long)c.x * 0xD2511F53u, b = (unsigned long long)c.z * 0xCD9E8D57u;
    c = make_uint4((unsigned)(b >> 32) ^ c.y ^ k0, (unsigned)b, (unsigned)(a >> 32) ^ c.w ^ k1, (unsigned)a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
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

// which of the eight columns of a group stay, a bit each.  Sixteen bits a column decide all but a tie with the
// threshold's upper half (one group in 8192); then the lower half is drawn too.
__device__ __forceinline__ unsigned kept8(const Drop& D, const DropKey& K, unsigned row, unsigned group) {
  const uint4 c = make_uint4(group, row, K.o0, K.o1);
  const uint4 w = philox(c, K.k0, K.k1);
  const unsigned word[4] = {w.x, w.y, w.z, w.w};
  unsigned keep = 0, tie = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const unsigned h = j & 1 ? word[j / 2] >> 16 : word[j / 2] & 0xffffu;
    keep |= (unsigned)(h >= D.threshold_hi) << j;
    tie |= (unsigned)(h == D.threshold_hi) << j;
  }
  if (tie != 0 && D.threshold_lo != 0) {
    const uint4 v = philox(make_uint4(c.x, c.y, c.z, c.w | 0x80000000u), K.k0, K.k1);
    const unsigned low[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const unsigned h = j & 1 ? low[j / 2] >> 16 : low[j / 2] & 0xffffu;
      if ((tie >> j & 1) && h < D.threshold_lo) keep &= ~(1u << j);
    }
  }
  return keep;
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
Drop to_drop(const lmg_dropout_spec* d);  // threshold_hi and _lo 0: nothing is dropped
inline bool drops(const Drop& D) { return D.threshold_hi != 0 || D.threshold_lo != 0; }
size_t embed_backward_bytes(unsigned rows, int ntypes, int width);
// f(T, O) for the element types of source and result, which agree or are float32 and 16 bits
template <class F>
cudaError_t by_vector_types(int in, int out, F f) {
  if (in == LMG_FLOAT32 && out == LMG_FLOAT32) return f(float(), float());
  if (in == LMG_FLOAT32 && out == LMG_BFLOAT16) return f(float(), __nv_bfloat16());
  if (in == LMG_FLOAT32 && out == LMG_FLOAT16) return f(float(), __half());
  if (in == LMG_BFLOAT16 && out == LMG_FLOAT32) return f(__nv_bfloat16(), float());
  if (in == LMG_FLOAT16 && out == LMG_FLOAT32) return f(__half(), float());
  if (in == LMG_BFLOAT16) return f(__nv_bfloat16(), __nv_bfloat16());
  return f(__half(), __half());
}
inline size_t element_bytes(int type) { return type == LMG_FLOAT32 ? 4 : 2; }
// rows of which any eight columns that begin at a multiple of eight lie on 16 bytes
inline bool rows_aligned(const lmg_vectors* v) {
  return reinterpret_cast<uintptr_t>(v->data) % 16 == 0 && v->ld * element_bytes(v->type) % 16 == 0;
}
inline size_t aligned256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace lmg

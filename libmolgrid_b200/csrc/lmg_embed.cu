// Type indices to rows of a table, and dropout.
#include "lmg_vectors.h"

#include <cmath>

namespace lmg {

int vectors_fail(int code, const char* msg) {
  lmg_internal_set_error(msg);
  return code;
}

int vectors_cuda(cudaError_t e, const char* what) {
  lmg_internal_set_error((std::string(what) + ": " + cudaGetErrorString(e)).c_str());
  return LMG_ERR_CUDA;
}

int check_slots(const lmg_slots* s, int width) {
  if (s == nullptr) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "null slots");
  if (s->batch < 0 || s->max_atoms < 0 || width < 0) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "negative size");
  if ((long long)s->batch * s->max_atoms >= 0x7fffffffll) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "2^31 slots and more");
  return LMG_OK;
}

int check_vectors(const lmg_vectors* v, int width, const char* name) {
  if (v == nullptr || v->data == nullptr)
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, (std::string(name) + " missing memory").c_str());
  if (v->type < LMG_FLOAT32 || v->type > LMG_FLOAT16)
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, (std::string(name) + " of unknown element type").c_str());
  if (v->ld < width) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, (std::string(name) + ": rows overlap").c_str());
  if (reinterpret_cast<uintptr_t>(v->data) % element_bytes(v->type) != 0)
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, (std::string(name) + " not aligned to its elements").c_str());
  return LMG_OK;
}

int check_drop(const lmg_dropout_spec* d) {
  if (d == nullptr) return LMG_OK;
  if (!(d->p >= 0.0 && d->p <= 1.0)) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "dropout probability outside [0, 1]");
  if (d->state == nullptr && d->offset >> 63) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "dropout offset of 2^63 and more");
  return LMG_OK;
}

int check_index(const lmg_slots* s, int ntypes) {
  if (ntypes < 0) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "negative size");
  if (s->index_type < LMG_INDEX_FLOAT32 || s->index_type > LMG_INDEX_INT64)
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "type indices of unknown element type");
  if (s->type_index == nullptr && s->batch > 0 && s->max_atoms > 0)
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "type indices missing memory");
  return LMG_OK;
}

Slots to_slots(const lmg_slots* s, int ntypes) {
  Slots S = {};
  S.rows = (unsigned)(s->batch * s->max_atoms);
  S.n = (unsigned)s->max_atoms;
  S.by_n = FastDiv(S.n ? S.n : 1);
  S.n_atoms = s->n_atoms;
  S.index = s->type_index;
  S.index_type = s->index_type;
  S.ntypes = ntypes;
  S.status = s->status;
  return S;
}

Drop to_drop(const lmg_dropout_spec* d) {
  Drop D = {};
  if (d == nullptr) return D;
  const unsigned long long t = (unsigned long long)std::llround(d->p * 4294967296.0);
  D.threshold_hi = (unsigned)(t >> 16);
  D.threshold_lo = (unsigned)(t & 0xffffu);
  D.scale = d->p < 1.0 ? (float)(1.0 / (1.0 - d->p)) : 0.f;
  D.seed = d->seed;
  D.offset = d->offset;
  D.state = d->state;
  return D;
}

namespace {

// A pass over rows first .. first + S.rows of a call, out[row][col] = scale * source row's value, dropped.  The source row is the
// slot's type's (LOOKUP) or the row itself.
struct RowArgs {
  Slots S;
  unsigned first, rows;
  int width;
  FastDiv by_groups, by_width;  // eight columns a group
  long long src_ld, out_ld;
  float scale;
  Drop D;
};

// Rows on 16 bytes: a thread takes groups of eight columns, which are one block of the generator, `UNITS` of them so that as many
// chains type -> row -> value are under way.
template <class T, class O, bool LOOKUP, bool DROP, int UNITS>
__global__ void __launch_bounds__(256) k_rows_aligned(RowArgs A, const T* src, O* out) {
  wait_for_stream();
  const DropKey K(A.D);
  const unsigned groups = A.by_groups.d, n = A.rows * groups, u0 = blockIdx.x * (256 * UNITS) + threadIdx.x;
  long long from[UNITS];
  unsigned row[UNITS];
  int col[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; k++) {
    const unsigned u = u0 + 256 * k;
    const unsigned r = A.by_groups(u < n ? u : 0);
    row[k] = A.first + r;
    col[k] = u < n ? (int)(u - r * groups) * 8 : A.width;  // behind the row's end: nothing is loaded or stored
    from[k] = row[k];
    if (LOOKUP) from[k] = slot_type(A.S, row[k]);
  }
  float v[UNITS][8];
#pragma unroll
  for (int k = 0; k < UNITS; k++) {
    if (!LOOKUP || from[k] >= 0) {
      load8<T, true>(src + from[k] * A.src_ld, col[k], A.width, v[k]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[k][i] = 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < UNITS; k++) {
    if (col[k] >= A.width) continue;
    const unsigned keep = DROP ? kept8(A.D, K, row[k], col[k] / 8) : 0xff;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (LOOKUP) v[k][i] *= A.scale;
      if (DROP) v[k][i] = keep >> i & 1 ? v[k][i] * A.D.scale : 0.f;
    }
    store8<O, true>(out + (long long)row[k] * A.out_ld, col[k], A.width, v[k]);
  }
}

// Rows of any width that follow one another without gaps, from 16 bytes on: a block writes 2048 values, 16 bytes a thread and
// turn, wherever rows begin and end in them; the types of its rows and the bits of its groups are made once, in shared memory.
constexpr int FLAT = 2048;

template <class T, class O, bool LOOKUP, bool DROP>
__global__ void __launch_bounds__(256) k_rows_flat(RowArgs A, const T* src, O* out) {
  __shared__ unsigned char kept[DROP ? FLAT + 8 : 1];
  __shared__ int types[LOOKUP ? FLAT + 8 : 1];
  wait_for_stream();
  const unsigned n = A.rows * (unsigned)A.width, e0 = blockIdx.x * FLAT, last = min(e0 + FLAT, n) - 1;
  const unsigned row0 = A.by_width(e0), row1 = A.by_width(last), groups = A.by_groups.d;
  if (LOOKUP)
    for (unsigned r = row0 + threadIdx.x; r <= row1; r += 256) types[r - row0] = slot_type(A.S, A.first + r);
  const unsigned g0 = row0 * groups + (e0 - row0 * A.width) / 8, g1 = row1 * groups + (last - row1 * A.width) / 8;
  if (DROP) {
    const DropKey K(A.D);
    for (unsigned g = g0 + threadIdx.x; g <= g1; g += 256) {
      const unsigned r = A.by_groups(g);
      kept[g - g0] = (unsigned char)kept8(A.D, K, A.first + r, g - r * groups);
    }
  }
  if (LOOKUP || DROP) __syncthreads();
  constexpr int N = 16 / sizeof(O);
#pragma unroll
  for (int j = 0; j < FLAT / 256 / N; j++) {
    const unsigned e = e0 + (j * 256 + threadIdx.x) * N;
    if (e > last) break;
    unsigned row = A.by_width(e), col = e - row * A.width;
    const bool whole = e + N <= n;
    float v[N];
    if (!LOOKUP && sizeof(T) == sizeof(O) && whole) {
      const uint4 a = *reinterpret_cast<const uint4*>(src + (long long)A.first * A.width + e);
      const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = to_float(h[i]);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (e + i < n) {
        if (LOOKUP) {
          const int t = types[row - row0];
          v[i] = t >= 0 ? to_float(src[t * A.src_ld + col]) * A.scale : 0.f;
        } else if (!whole) {
          v[i] = to_float(src[(long long)A.first * A.width + e + i]);
        }
        if (DROP) v[i] = kept[row * groups + col / 8 - g0] >> (col & 7) & 1 ? v[i] * A.D.scale : 0.f;
        if (++col == (unsigned)A.width) col = 0, row++;
      }
    }
    O* to = out + (long long)A.first * A.width + e;
    if (whole) {
      uint4 a;
      O* h = reinterpret_cast<O*>(&a);
#pragma unroll
      for (int i = 0; i < N; i++) h[i] = from_float<O>(v[i]);
      *reinterpret_cast<uint4*>(to) = a;
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (e + i < n) to[i] = from_float<O>(v[i]);
    }
  }
}

// everything else: a thread a value
template <class T, class O, bool LOOKUP>
__global__ void __launch_bounds__(256) k_rows(RowArgs A, const T* src, O* out, bool dropping) {
  wait_for_stream();
  const DropKey K(A.D);
  const long long n = (long long)A.rows * A.width;
  for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (long long)gridDim.x * blockDim.x) {
    const unsigned r = (unsigned)(e / A.width), col = (unsigned)(e - (long long)r * A.width), row = A.first + r;
    long long from = row;
    if (LOOKUP) from = slot_type(A.S, row);  // an int: -1 stays negative
    float v = 0.f;
    if (from >= 0) v = to_float(src[from * A.src_ld + col]) * A.scale;
    if (dropping) v = kept8(A.D, K, row, col / 8) >> (col & 7) & 1 ? v * A.D.scale : 0.f;
    out[(long long)row * A.out_ld + col] = from_float<O>(v);
  }
}

__global__ void k_next_draw(unsigned long long* state, unsigned long long* taken) {
  wait_for_stream();
  const unsigned long long offset = state[1];
  taken[0] = state[0];
  taken[1] = offset;
  state[1] = (offset + 1) & 0x7fffffffffffffffull;
}

template <bool LOOKUP>
cudaError_t launch_rows(const Slots& S, const lmg_vectors* src, const lmg_vectors* out, int width, float scale, const Drop& D, long* launches,
                        cudaStream_t st) {
  RowArgs A = {S, 0, S.rows, width, FastDiv((unsigned)((long long)width + 7 >> 3)), FastDiv((unsigned)width), src->ld, out->ld, scale, D};
  const bool aligned = rows_aligned(src) && rows_aligned(out);
  const bool flat = out->ld == width && reinterpret_cast<uintptr_t>(out->data) % 16 == 0 &&
                    (LOOKUP || (src->ld == width && reinterpret_cast<uintptr_t>(src->data) % 16 == 0));
  // passes of less than 2^30 values, a multiple of eight rows so that each begins on 16 bytes again
  const unsigned most = width > 1 << 26 ? 0 : (1u << 30) / (unsigned)width & ~7u;
  return by_vector_types(src->type, out->type, [&](auto t, auto o) {
    typedef decltype(t) T;
    typedef decltype(o) O;
    const T* from = static_cast<const T*>(src->data);
    O* to = static_cast<O*>(out->data);
    cudaError_t e = cudaSuccess;
    if ((!aligned && !flat) || most == 0) {
      const long long blocks = ((long long)S.rows * width + 255) / 256;
      ++*launches;
      return launch_early(k_rows<T, O, LOOKUP>, dim3((unsigned)(blocks < 148 * 64 ? blocks : 148 * 64)), 256, 0, st, A, from, to, drops(D));
    }
    for (A.first = 0; A.first < S.rows && e == cudaSuccess; A.first += A.rows) {
      A.rows = S.rows - A.first < most ? S.rows - A.first : most;
      const unsigned units = A.rows * A.by_groups.d;
      ++*launches;
      if (!aligned) {
        e = launch_early(drops(D) ? k_rows_flat<T, O, LOOKUP, true> : k_rows_flat<T, O, LOOKUP, false>,
                         dim3((unsigned)(((long long)A.rows * width + FLAT - 1) / FLAT)), 256, 0, st, A, from, to);
      } else if (units <= 148 * 256 * 4) {  // one wave: more threads instead of more units a thread
        e = launch_early(drops(D) ? k_rows_aligned<T, O, LOOKUP, true, 1> : k_rows_aligned<T, O, LOOKUP, false, 1>, dim3((units + 255) / 256), 256, 0, st,
                         A, from, to);
      } else {
        e = launch_early(drops(D) ? k_rows_aligned<T, O, LOOKUP, true, 4> : k_rows_aligned<T, O, LOOKUP, false, 4>, dim3((units + 1023) / 1024), 256, 0, st,
                         A, from, to);
      }
    }
    return e;
  });
}

}  // namespace
}  // namespace lmg

extern "C" {

int lmg_embed_types(const lmg_slots* slots, int ntypes, int width, const lmg_vectors* table, float scale,
                    const lmg_dropout_spec* drop, const lmg_vectors* out, void* stream) {
  using namespace lmg;
  int rc;
  if ((rc = check_slots(slots, width)) || (rc = check_index(slots, ntypes)) || (rc = check_drop(drop))) return rc;
  if (slots->batch == 0 || slots->max_atoms == 0 || width == 0) return LMG_OK;
  if ((rc = check_vectors(out, width, "output"))) return rc;
  lmg_vectors none = *out;  // a table without types is not read
  none.ld = width;
  if (ntypes == 0) table = &none;
  if ((rc = check_vectors(table, width, "table"))) return rc;
  if (table->type != out->type && table->type != LMG_FLOAT32)
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "table and output differ in type, and the table is not float32");
  long launches = 0;
  const cudaError_t e = launch_rows<true>(to_slots(slots, ntypes), table, out, width, scale, to_drop(drop), &launches, (cudaStream_t)stream);
  lmg_internal_count_launches(launches);
  if (e != cudaSuccess) return vectors_cuda(e, "looking up types");
  return LMG_OK;
}

int lmg_dropout(int rows, int width, const lmg_vectors* x, const lmg_dropout_spec* drop, const lmg_vectors* out, void* stream) {
  using namespace lmg;
  lmg_slots s = {};
  s.batch = 1;
  s.max_atoms = rows;
  int rc;
  if ((rc = check_slots(&s, width)) || (rc = check_drop(drop))) return rc;
  if (drop == nullptr) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "null dropout");
  if (rows == 0 || width == 0) return LMG_OK;
  if ((rc = check_vectors(x, width, "input")) || (rc = check_vectors(out, width, "output"))) return rc;
  if (x->type != out->type) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "input and output differ in type");
  long launches = 0;
  const cudaError_t e = launch_rows<false>(to_slots(&s, 0), x, out, width, 1.f, to_drop(drop), &launches, (cudaStream_t)stream);
  lmg_internal_count_launches(launches);
  if (e != cudaSuccess) return vectors_cuda(e, "dropping values");
  return LMG_OK;
}

int lmg_dropout_next(unsigned long long* state, unsigned long long* taken, void* stream) {
  if (state == nullptr || taken == nullptr) return lmg::vectors_fail(LMG_ERR_INVALID_ARGUMENT, "generator state missing memory");
  const cudaError_t e = lmg::launch_early(lmg::k_next_draw, dim3(1), 1, 0, (cudaStream_t)stream, state, taken);
  if (e != cudaSuccess) return lmg::vectors_cuda(e, "taking a draw");
  lmg_internal_count_launches(1);
  return LMG_OK;
}

}  // extern "C"

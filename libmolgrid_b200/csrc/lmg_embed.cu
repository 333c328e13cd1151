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

cudaError_t allow_smem_of(const void* kernel) {
  struct Asked {
    const void* kernel;
    int device;
  };
  static thread_local Asked asked[64] = {};
  int device = -1;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  Asked& a = asked[(reinterpret_cast<uintptr_t>(kernel) >> 4) % 64];
  if (a.kernel == kernel && a.device == device) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MOST);
  if (e == cudaSuccess) a = {kernel, device};
  return e;
}

int check_slots(const lmg_slots* s, int width) {
  if (s == nullptr) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "null slots");
  if (s->batch < 0 || s->max_atoms < 0 || width < 0) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "negative size");
  if ((long long)s->batch * s->max_atoms >= 0x7fffffffll) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "2^31 slots and more");
  if (width >= 1 << 30) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "2^30 columns and more");
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
  D.upper = t >> 32 ? 65535u : (unsigned)(t >> 16);
  D.lower = t >> 32 ? 65536u : (unsigned)(t & 0xffffu);
  D.scale = d->p < 1.0 ? (float)(1.0 / (1.0 - d->p)) : 0.f;
  D.seed = d->seed;
  D.offset = d->offset;
  D.state = d->state;
  return D;
}

namespace {

// A pass over rows first .. first + rows of a call, out[row][col] = scale * source row's value, dropped.  The source row is the
// slot's type's (LOOKUP) or the row itself.
struct RowArgs {
  Slots S;
  unsigned first, rows;
  int width;
  unsigned groups, across, down;             // of eight columns a row; a block has `across` x `down` threads at work
  FastDiv by_groups, by_width, by_across;
  long long src_ld, out_ld;
  float scale;
  Drop D;
};

// Rows on 16 bytes: a thread takes COLS columns of UNITS rows, so that as many loads are under way; with dropout eight columns, which are one
// block of the generator.  The types of a block's rows are looked up once, in shared memory.
constexpr int UNITS_MOST = 4;

template <class T, class O, bool LOOKUP, bool DROP, int COLS, int UNITS>
__global__ void __launch_bounds__(256, DROP && UNITS == UNITS_MOST ? 5 : 6) k_rows_aligned(RowArgs A, const T* src, O* out) {
  __shared__ int types[LOOKUP ? 256 * UNITS : 1];
  wait_for_stream();
  const unsigned first = blockIdx.x * (A.down * UNITS);
  if (LOOKUP) {
    for (unsigned i0 = threadIdx.x; i0 < A.down * UNITS; i0 += blockDim.x * UNITS) {
      unsigned r[UNITS];
      bool in[UNITS];
      int t[UNITS];
#pragma unroll
      for (int k = 0; k < UNITS; k++) {
        const unsigned i = i0 + k * blockDim.x;
        r[k] = A.first + first + i;
        in[k] = i < A.down * UNITS && first + i < A.rows;
      }
      slot_types(A.S, r, in, t);
#pragma unroll
      for (int k = 0; k < UNITS; k++)
        if (i0 + k * blockDim.x < A.down * UNITS) types[i0 + k * blockDim.x] = t[k];
    }
    __syncthreads();
  }
  const unsigned sub = A.by_across(threadIdx.x), g = blockIdx.y * A.across + threadIdx.x - sub * A.across;
  if (sub >= A.down || g >= A.groups) return;
  const int col = (int)g * COLS;
  Raw<T, COLS> raw[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; k++) {
    const unsigned i = sub + k * A.down;
    const int type = LOOKUP ? types[i] : 0;
    if (LOOKUP ? type >= 0 : first + i < A.rows) raw[k].load(src + (LOOKUP ? (long long)type : (long long)(A.first + first + i)) * A.src_ld, col, A.width);
    else raw[k].clear();
  }
  const unsigned row = A.first + first + sub;
  uint4 c[UNITS];
  const DropKey K(A.D);
  if (DROP) {
#pragma unroll
    for (int k = 0; k < UNITS; k++) c[k] = make_uint4(g, row + k * A.down, K.o0, K.o1);
    philox(c, K.k0, K.k1);
  }
#pragma unroll
  for (int k = 0; k < UNITS; k++) {
    if (first + sub + k * A.down >= A.rows) break;
    float v[COLS];
#pragma unroll
    for (int i = 0; i < COLS; i++) v[i] = LOOKUP ? raw[k].get(i) * A.scale : raw[k].get(i);
    if constexpr (DROP) {
      Bits8 b;
      b.set(c[k], A.D, K, row + k * A.down, g);
      b.apply(A.D.scale, v);
    }
    store_cols<O, COLS>(out + (long long)(row + k * A.down) * A.out_ld, col, A.width, v);
  }
}

// Rows of any width that follow one another without gaps, from 16 bytes on: a block writes eight values a thread, 16 bytes a thread and
// turn (with 4 bytes 8476 looked up rows of 3005 bfloat16 take 61 us instead of 54), wherever rows begin and end in them.  The types of its rows, and which of its values stay, a bit each, are made once,
// in shared memory.
template <class T, class O, bool LOOKUP, bool DROP, int THREADS>
__global__ void __launch_bounds__(THREADS, (DROP ? 1280 : 1536) / THREADS) k_rows_flat(RowArgs A, const T* src, O* out) {
  constexpr int FLAT = 8 * THREADS;
  __shared__ unsigned kept[DROP ? FLAT / 32 : 1];
  __shared__ int types[LOOKUP ? FLAT : 1];
  const unsigned n = A.rows * (unsigned)A.width, e0 = blockIdx.x * FLAT, end = min(e0 + FLAT, n);
  const unsigned row0 = A.by_width(e0), row1 = A.by_width(end - 1), groups = A.by_groups.d;
  if (DROP) {
    for (int i = threadIdx.x; i < FLAT / 32; i += THREADS) kept[i] = 0;
    __syncthreads();
  }
  wait_for_stream();
  constexpr int N = 16 / (int)sizeof(O), TURNS = 8 / N;
  const T* from = src + (LOOKUP ? 0 : (long long)A.first * A.width);
  O* to = out + (long long)A.first * A.width;
  Raw<T, LOOKUP ? 4 : N> raw[LOOKUP ? 1 : TURNS];  // on their way while the bits are made
  if constexpr (!LOOKUP) {
#pragma unroll
    for (int j = 0; j < TURNS; j++) {
      const unsigned e = e0 + (j * THREADS + threadIdx.x) * N;
      if (e < end) raw[j].load(from + e, 0, (int)min(end - e, (unsigned)N));
    }
  }
  if (LOOKUP)
    for (unsigned r0 = row0 + threadIdx.x; r0 <= row1; r0 += 4 * THREADS) {  // four at a time are on their way
      unsigned r[4];
      bool in[4];
      int t[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        r[k] = A.first + r0 + k * THREADS;
        in[k] = r0 + k * THREADS <= row1;
      }
      slot_types(A.S, r, in, t);
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (in[k]) types[r0 + k * THREADS - row0] = t[k];
    }
  if (DROP) {
    const DropKey K(A.D);
    const unsigned g0 = row0 * groups + (e0 - row0 * A.width) / 8, g1 = row1 * groups + (end - 1 - row1 * A.width) / 8;
    for (unsigned g = g0 + threadIdx.x; g <= g1; g += THREADS) {
      const unsigned r = A.by_groups(g), in_row = g - r * groups;
      unsigned bits = kept8(A.D, K, A.first + r, in_row);
      if ((in_row + 1) * 8 > (unsigned)A.width) bits &= (1u << (A.width & 7)) - 1;
      // the group's first value may lie before the block's, its last behind it
      const int at = (int)(r * (unsigned)A.width + in_row * 8 - e0);
      const unsigned long long wide = (unsigned long long)bits << (at & 31);
      const int word = at >> 5;  // -1: the bits that reach into word 0 are those of the upper half
      if (word >= 0 && (unsigned)wide != 0) atomicOr(&kept[word], (unsigned)wide);
      if (word + 1 < FLAT / 32 && (unsigned)(wide >> 32) != 0) atomicOr(&kept[word + 1], (unsigned)(wide >> 32));
    }
  }
  if (LOOKUP || DROP) __syncthreads();
#pragma unroll
  for (int j = 0; j < TURNS; j++) {
    const unsigned e = e0 + (j * THREADS + threadIdx.x) * N;
    if (e >= end) break;
    const bool whole = e + N <= end;
    float v[N];
    if constexpr (LOOKUP) {
      unsigned row = A.by_width(e), col = e - row * A.width;
      if (col + N <= (unsigned)A.width) {  // within a row
        const int t = types[row - row0];
        const T* p = from + t * A.src_ld + col;
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = t >= 0 ? to_float(p[i]) * A.scale : 0.f;
      } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
          if (e + i >= end) break;
          const int t = types[row - row0];
          v[i] = t >= 0 ? to_float(from[t * A.src_ld + col]) * A.scale : 0.f;
          if (++col == (unsigned)A.width) col = 0, row++;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = raw[j].get(i);
    }
    if (DROP) {
      const unsigned bits = kept[(e - e0) / 32] >> ((e - e0) & 31);
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = bits >> i & 1 ? v[i] * A.D.scale : 0.f;
    }
    if (whole) {
      store_cols<O, N>(to + e, 0, N, v);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (e + i < end) to[e + i] = from_float<O>(v[i]);
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
  const unsigned eights = (unsigned)(((long long)width + 7) >> 3);
  RowArgs A = {S, 0, S.rows, width, eights, 0, 0, FastDiv(eights), FastDiv((unsigned)width), FastDiv(), src->ld, out->ld, scale, D};
  const bool aligned = rows_aligned(src) && rows_aligned(out);
  const bool flat = out->ld == width && reinterpret_cast<uintptr_t>(out->data) % 16 == 0 &&
                    (LOOKUP || (src->ld == width && reinterpret_cast<uintptr_t>(src->data) % 16 == 0));
  // passes of less than 2^30 values, a multiple of eight rows so that each begins on 16 bytes again; wider rows would be more than the 65535
  // tiles of 256 groups of four columns that a launch has
  const unsigned most = width > 65535 * 1024 ? 0 : (1u << 30) / (unsigned)width & ~7u;
  return by_vector_types<LOOKUP, false>(src->type, out->type, [&](auto t, auto o) {
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
      ++*launches;
      if (!aligned) {
        // few values: more blocks of fewer threads, which wait for fewer draws
        const long long n = (long long)A.rows * width;
        const int threads = n <= 148 * 2048 ? 64 : 256;
        auto kernel = drops(D) ? k_rows_flat<T, O, LOOKUP, true, 256> : k_rows_flat<T, O, LOOKUP, false, 256>;
        if (threads == 64) kernel = drops(D) ? k_rows_flat<T, O, LOOKUP, true, 64> : k_rows_flat<T, O, LOOKUP, false, 64>;
        e = launch_early(kernel, dim3((unsigned)((n + 8 * threads - 1) / (8 * threads))), threads, 0, st, A, from, to);
        continue;
      }
      // 16 bytes a thread of whatever is wider; dropout goes by eights
      const bool fours = !drops(D) && (sizeof(T) == 4 || sizeof(O) == 4);
      A.groups = fours ? (unsigned)(width + 3) / 4 : eights;
      const unsigned tiles = (A.groups + 255) / 256;
      A.across = (A.groups + tiles - 1) / tiles;
      A.down = 256 / A.across;
      A.by_across = FastDiv(A.across);
      // few rows: more threads instead of more rows a thread
      constexpr int DRAWS = sizeof(T) == 2 ? UNITS_MOST : 2;  // of a thread side by side, as far as registers go: 26.6 and 25.3 us for 8192 x 4096 bfloat16
      const int units = (size_t)A.rows * A.groups <= 148 * 512 ? 1 : drops(D) ? DRAWS : UNITS_MOST;
      const dim3 grid((A.rows + A.down * units - 1) / (A.down * units), tiles);
      const unsigned threads = (A.across * A.down + 31) / 32 * 32;
      auto kernel = units == 1 ? k_rows_aligned<T, O, LOOKUP, true, 8, 1> : k_rows_aligned<T, O, LOOKUP, true, 8, DRAWS>;
      if (fours) kernel = units == 1 ? k_rows_aligned<T, O, LOOKUP, false, 4, 1> : k_rows_aligned<T, O, LOOKUP, false, 4, UNITS_MOST>;
      else if (!drops(D)) kernel = units == 1 ? k_rows_aligned<T, O, LOOKUP, false, 8, 1> : k_rows_aligned<T, O, LOOKUP, false, 8, UNITS_MOST>;
      e = launch_early(kernel, grid, threads, 0, st, A, from, to);
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

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

// out[row][col] = scale * source row's value, dropped.  LOOKUP: the source row is the slot's type's, else the row itself.
template <class T, class O, bool LOOKUP>
__global__ void __launch_bounds__(256) k_rows(Slots S, const T* src, long long src_ld, O* out, long long out_ld, int width,
                                              float scale, bool dropping, Drop D) {
  wait_for_stream();
  const DropKey K(D);
  const long long n = (long long)S.rows * width;
  for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (long long)gridDim.x * blockDim.x) {
    const unsigned row = (unsigned)(e / width), col = (unsigned)(e - (long long)row * width);
    long long from = row;
    if (LOOKUP) from = slot_type(S, row);  // an int: -1 stays negative
    float v = 0.f;
    if (from >= 0) v = to_float(src[from * src_ld + col]) * scale;
    if (dropping) v = kept8(D, K, row, col / 8) >> (col & 7) & 1 ? v * D.scale : 0.f;
    out[(long long)row * out_ld + col] = from_float<O>(v);
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
cudaError_t launch_rows(const Slots& S, const lmg_vectors* src, const lmg_vectors* out, int width, float scale, const Drop& D,
                        cudaStream_t st) {
  const long long blocks = ((long long)S.rows * width + 255) / 256;
  const dim3 grid((unsigned)(blocks < 148 * 64 ? blocks : 148 * 64));
  return by_vector_types(src->type, out->type, [&](auto t, auto o) {
    return launch_early(k_rows<decltype(t), decltype(o), LOOKUP>, grid, 256, 0, st, S, static_cast<const decltype(t)*>(src->data), src->ld,
                        static_cast<decltype(o)*>(out->data), out->ld, width, scale, drops(D), D);
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
  const cudaError_t e = launch_rows<true>(to_slots(slots, ntypes), table, out, width, scale, to_drop(drop), (cudaStream_t)stream);
  if (e != cudaSuccess) return vectors_cuda(e, "looking up types");
  lmg_internal_count_launches(1);
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
  const cudaError_t e = launch_rows<false>(to_slots(&s, 0), x, out, width, 1.f, to_drop(drop), (cudaStream_t)stream);
  if (e != cudaSuccess) return vectors_cuda(e, "dropping values");
  lmg_internal_count_launches(1);
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

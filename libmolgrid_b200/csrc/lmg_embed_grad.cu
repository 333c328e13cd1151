// Gradient of a table of type vectors: for each type the sum of its slots' gradients.
//
// Few types, many slots each (k_type_tables): a warp keeps a table of its own in shared memory and adds row after row to
// it, so the gradients are read once, in order; the blocks' tables are summed afterwards.  Otherwise the slots are sorted by
// type, and groups of lanes walk equal pieces of the sorted slots: a type that lies within a piece is written at once, one that
// crosses pieces is put together from partial sums.  In one launch where each block can find its own slots among few
// (k_type_small) or types are shared out among clusters (k_type_ranges), else by a stable radix sort (k_sort_cluster, or
// k_sort_count and k_sort_move), k_type_pieces and k_type_joins.  Equal pieces, not types, because a type can hold one slot or all of them.  No atomics touch
// a sum: its order is fixed by the sizes alone.
#include "lmg_vectors.h"

namespace lmg {
namespace {

// ---- few types --------------------------------------------------------------------------------------------------------
constexpr int TABLE_COLS = 32, TABLE_LANES = 8;  // columns of a table, lanes that share a row: four columns each

// A warp takes 32 consecutive slots at a time, four side by side: eight lanes with a table of their own, which nobody else touches, add
// them to it one after the other.  parts[block][type][width], or `grad` where one block does all.  (A lane a column and a
// table a warp instead took 33 instructions a slot and 16 us for 200000 slots of 28.)
template <class T, class O, bool VEC, bool DROP>
__global__ void __launch_bounds__(512) k_type_tables(Slots S, unsigned per, const T* diff, long long diff_ld, int width, float* parts, O* grad,
                                                     long long grad_ld, float scale, Drop D) {
  extern __shared__ float4 tables[];  // [warp][4][type][8]
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32, warps = blockDim.x / 32, V = S.ntypes, q = lane / TABLE_LANES, l = lane % TABLE_LANES;
  for (int i = threadIdx.x; i < warps * 4 * V * TABLE_LANES; i += blockDim.x) tables[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  wait_for_stream();
  if (gridDim.x > 1) no_status(parts);
  const DropKey K(D);
  float4* mine = tables + (size_t)(warp * 4 + q) * V * TABLE_LANES + l;
  const int col = blockIdx.y * TABLE_COLS + l * 4;
  const unsigned long long at = (unsigned long long)(blockIdx.x * warps + warp) * per;
  const unsigned begin = at < S.rows ? (unsigned)at : S.rows, end = S.rows - begin < per ? S.rows : begin + per;
  // types two turns ahead, values one
  auto types = [&](unsigned r0) { return r0 < end && end - r0 > lane ? slot_type(S, r0 + lane) : -1; };
  int t[8], t_next[8];
  Raw<T, 4, VEC> raw[8], raw_next[8];
  auto fetch = [&](unsigned r0, int type, int (&to_t)[8], Raw<T, 4, VEC> (&to_v)[8]) {
    const T* from = diff + (long long)(r0 + q) * diff_ld;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      to_t[j] = __shfl_sync(0xffffffffu, type, j * 4 + q);
      if (col >= width) to_t[j] = -1;
      if (to_t[j] >= 0) to_v[j].load(from + j * 4 * diff_ld, col, width);
    }
  };
  fetch(begin, types(begin), t, raw);
  int type_next = types(begin + 32);
  __syncthreads();
  for (unsigned r0 = begin; r0 < end; r0 += 32) {
    fetch(r0 + 32, type_next, t_next, raw_next);
    type_next = types(r0 + 64);
    unsigned keep[8];
    if (DROP) {
      // eight slots of four groups of eight columns a turn: a lane draws for one of them and hands its bits round
      const unsigned group = blockIdx.y * (TABLE_COLS / 8) + lane % 4;
      uint4 c[4];
#pragma unroll
      for (int j = 0; j < 4; j++) c[j] = make_uint4(group, r0 + j * 8 + lane / 4, K.o0, K.o1);
      philox(c, K.k0, K.k1);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        Bits8 b;
        b.set(c[j], D, K, r0 + j * 8 + lane / 4, group);
        const unsigned bits = b.mask();
#pragma unroll
        for (int h = 0; h < 2; h++) keep[2 * j + h] = __shfl_sync(0xffffffffu, bits, (h * 4 + q) * 4 + l / 2) >> (l & 1) * 4;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (t[j] >= 0) {
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = DROP ? (keep[j] >> c & 1 ? raw[j].get(c) * D.scale : 0.f) : raw[j].get(c);
        float4* to = mine + t[j] * TABLE_LANES;
        float4 s = *to;
        s.x += v[0], s.y += v[1], s.z += v[2], s.w += v[3];
        *to = s;
      }
      t[j] = t_next[j];
      raw[j] = raw_next[j];
    }
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(tables);
  for (int i = threadIdx.x; i < V * TABLE_COLS; i += blockDim.x) {
    const int c = blockIdx.y * TABLE_COLS + (i & (TABLE_COLS - 1)), type = i / TABLE_COLS;
    if (c >= width) continue;
    float sum = 0.f;
#pragma unroll 8
    for (int w = 0; w < warps * 4; w++) sum += all[(size_t)w * V * TABLE_COLS + i];
    if (gridDim.x == 1) grad[(long long)type * grad_ld + c] = from_float<O>(sum * scale);
    else parts[((size_t)blockIdx.x * V + type) * width + c] = sum;
  }
}

// the sum of all blocks' tables: 32 values a block, 32 threads a value
template <class O>
__global__ void __launch_bounds__(1024) k_table_sums(const float* parts, int n, int V, int width, O* grad, long long grad_ld, float scale) {
  __shared__ float s[32][33];
  wait_for_stream();
  const size_t M = (size_t)V * width, first = (size_t)blockIdx.x * 32;
  const int lane = threadIdx.x & 31, slice = threadIdx.x / 32;
  float sum = 0.f;
  if (first + lane < M) {
#pragma unroll 8
    for (int p = slice; p < n; p += 32) sum += parts[p * M + first + lane];
  }
  s[slice][lane] = sum;
  __syncthreads();
  sum = s[lane][slice];  // a warp a value
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const size_t o = first + slice;
  if (lane == 0 && o < M) grad[(long long)(o / width) * grad_ld + o % width] = from_float<O>(sum * scale);
}

// ---- the sort ---------------------------------------------------------------------------------------------------------
constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, SORT_TILE_MOST = 32768, SORT_BITS_MOST = 11;

// what a launch of the sort clears on the way: a share of the table's gradient, with what is idle beside the tiles
struct Clear {
  char* p;       // on a boundary of 16 bytes
  size_t bytes;  // even
};

struct SortArgs {
  Slots S;
  unsigned tiles, tile;  // tiles of `tile` slots, a multiple of SORT_THREADS
  int shift, bits;
  const unsigned *key_in, *row_in;  // null in the first pass, which reads the types themselves
  unsigned *key_out, *row_out;
  unsigned* counts;  // [tiles][1 << bits]
  Clear clear;
};

__device__ __forceinline__ unsigned sort_key(const SortArgs& A, unsigned i) {
  if (A.key_in != nullptr) return A.key_in[i];
  const int t = slot_type(A.S, i);
  return t < 0 ? (unsigned)A.S.ntypes : (unsigned)t;  // empty slots come last
}

__device__ void clear_share(const Clear& C, unsigned block, unsigned blocks) {
  uint4* p = reinterpret_cast<uint4*>(C.p);
  for (size_t i = (size_t)block * SORT_THREADS + threadIdx.x; i < C.bytes / 16; i += (size_t)blocks * SORT_THREADS) p[i] = make_uint4(0, 0, 0, 0);
  if (block == 0 && threadIdx.x < C.bytes % 16 / 2) reinterpret_cast<unsigned short*>(C.p + C.bytes / 16 * 16)[threadIdx.x] = 0;
}

// The lanes whose digit of `bits` bits is this lane's, among those with a slot.  A ballot a bit:
// __match_any_sync took no less, about 1100 cycles a turn of 32 warps.
__device__ __forceinline__ unsigned same_digit(unsigned digit, int bits, bool slot) {
  unsigned same = __ballot_sync(0xffffffffu, slot);
  for (int b = 0; b < bits; b++) {
    const bool set = digit >> b & 1;
    const unsigned with = __ballot_sync(0xffffffffu, set);
    same &= set ? with : ~with;
  }
  return same;
}

__global__ void __launch_bounds__(SORT_THREADS) k_sort_count(SortArgs A) {
  __shared__ unsigned count[1 << SORT_BITS_MOST];
  wait_for_stream();
  if (A.key_in == nullptr) no_status(A.key_out);
  if (blockIdx.x >= A.tiles) return clear_share(A.clear, blockIdx.x - A.tiles, gridDim.x - A.tiles);
  const unsigned bins = 1u << A.bits;
  for (unsigned b = threadIdx.x; b < bins; b += SORT_THREADS) count[b] = 0;
  __syncthreads();
  const unsigned begin = blockIdx.x * A.tile, end = min(begin + A.tile, A.S.rows);
  for (unsigned i = begin + threadIdx.x; i < end; i += SORT_THREADS) atomicAdd(&count[sort_key(A, i) >> A.shift & (bins - 1)], 1u);
  __syncthreads();
  for (unsigned b = threadIdx.x; b < bins; b += SORT_THREADS) A.counts[(size_t)blockIdx.x * bins + b] = count[b];
}

// Places of a tile's slots: behind all slots of smaller digits, and those of the same digit in tiles, warps and lanes before.
__global__ void __launch_bounds__(SORT_THREADS) k_sort_move(SortArgs A) {
  extern __shared__ unsigned sort_shared[];
  wait_for_stream();
  if (blockIdx.x >= A.tiles) return clear_share(A.clear, blockIdx.x - A.tiles, gridDim.x - A.tiles);
  const unsigned bins = 1u << A.bits, mask = bins - 1, tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  unsigned* base = sort_shared;                                                         // [bins] first place of a digit's slots here
  unsigned* total = base + bins;                                                      // [slices][bins]
  const unsigned slices = bins < SORT_THREADS ? SORT_THREADS / bins : 1;
  unsigned* before = total + slices * bins;                                           // [slices][bins]
  unsigned short* mine = reinterpret_cast<unsigned short*>(before + slices * bins) + warp * bins;  // [warps][bins]
  for (unsigned b = tid; b < slices * bins; b += SORT_THREADS) {
    unsigned all = 0, earlier = 0;
#pragma unroll 8
    for (unsigned t = b / bins; t < A.tiles; t += slices) {
      const unsigned n = A.counts[(size_t)t * bins + (b & mask)];
      all += n;
      earlier += t < blockIdx.x ? n : 0;
    }
    total[b] = all;
    before[b] = earlier;
  }
  for (unsigned b = lane; b < bins; b += 32) mine[b] = 0;
  __syncthreads();
  // digits' totals to their first places; a thread has two digits at most
  __shared__ unsigned warp_sum[SORT_WARPS];
  unsigned sum[2] = {0, 0}, off[2] = {0, 0};
  const unsigned b0 = bins > SORT_THREADS ? 2 * tid : tid, nb = bins > SORT_THREADS ? 2 : b0 < bins ? 1 : 0;
  for (unsigned k = 0; k < nb; k++)
    for (unsigned s = 0; s < slices; s++) {
      sum[k] += total[s * bins + b0 + k];
      off[k] += before[s * bins + b0 + k];
    }
  unsigned run = sum[0] + sum[1];
  for (unsigned o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) warp_sum[warp] = run;
  __syncthreads();
  unsigned first = run - sum[0] - sum[1];
  for (unsigned w = 0; w < warp; w++) first += warp_sum[w];
  if (nb > 0) base[b0] = first + off[0];
  if (nb > 1) base[b0 + 1] = first + sum[0] + off[1];
  // how many of each digit every warp has
  const unsigned per = A.tile / SORT_WARPS, begin = blockIdx.x * A.tile + warp * per, end = min(begin + per, A.S.rows);
  for (unsigned i0 = begin; i0 < end; i0 += 32) {
    const unsigned i = i0 + lane, d = i < end ? sort_key(A, i) >> A.shift & mask : 0;
    const unsigned peers = same_digit(d, A.bits, i < end);
    if (i < end && (peers & ((1u << lane) - 1)) == 0) mine[d] += (unsigned short)__popc(peers);
    __syncwarp();
  }
  __syncthreads();
  unsigned short* all = reinterpret_cast<unsigned short*>(before + slices * bins);
  for (unsigned b = tid; b < bins; b += SORT_THREADS) {
    unsigned at = 0;
    for (unsigned w = 0; w < SORT_WARPS; w++) {
      const unsigned n = all[w * bins + b];
      all[w * bins + b] = (unsigned short)at;
      at += n;
    }
  }
  __syncthreads();
  for (unsigned i0 = begin; i0 < end; i0 += 32) {
    const unsigned i = i0 + lane, key = i < end ? sort_key(A, i) : 0, d = key >> A.shift & mask;
    const unsigned peers = same_digit(d, A.bits, i < end), lower = peers & ((1u << lane) - 1);
    const unsigned at = i < end ? base[d] + mine[d] + __popc(lower) : ~0u;
    __syncwarp();
    if (i < end && lower == 0) mine[d] += (unsigned short)__popc(peers);
    __syncwarp();
    if (at < A.S.rows) {  // always, for types that nobody changes meanwhile
      A.key_out[at] = key;
      A.row_out[at] = A.row_in != nullptr ? A.row_in[i] : i;
    }
  }
}

// ---- the sort of up to 32768 slots, in one launch -----------------------------------------------------------------------------
// Eight blocks of a cluster hold an eighth of the slots each, four a thread, and read one another's counts in shared memory; the
// other clusters of the launch clear the table's gradient meanwhile.  (Gradients with two launches a
// pass: 25551 slots of 350 types 30 us instead of 20.7, 16384 of 50021 types and 1024 bfloat16 49 instead of 42.5.)
constexpr unsigned CLUSTER = 8, CLUSTER_KEYS = 4;
constexpr int CLUSTER_BITS_MOST = 10;
static_assert(1 << CLUSTER_BITS_MOST <= SORT_THREADS, "a thread has one digit");

struct ClusterSortArgs {
  Slots S;
  unsigned each;            // slots of a block, a multiple of SORT_THREADS
  int passes, bits;
  unsigned *key[2], *row[2];
  Clear clear;
};

__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();  // a warp arrives as one, and waits as one
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// what another block of the cluster has at the same place in its shared memory
__device__ __forceinline__ unsigned cluster_load(const unsigned* p, unsigned rank) {
  unsigned v;
  const unsigned at = (unsigned)__cvta_generic_to_shared(p);
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}" : "=r"(v) : "r"(at), "r"(rank) : "memory");
  return v;
}

__global__ void __launch_bounds__(SORT_THREADS) k_sort_cluster(ClusterSortArgs A) {
  extern __shared__ unsigned sort_shared[];
  __shared__ unsigned warp_sum[SORT_WARPS];
  wait_for_stream();
  no_status(A.key[0]);
  if (blockIdx.x >= CLUSTER) return clear_share(A.clear, blockIdx.x - CLUSTER, gridDim.x - CLUSTER);
  const unsigned bins = 1u << A.bits, mask = bins - 1, tid = threadIdx.x, lane = tid & 31, warp = tid / 32, block = blockIdx.x;
  unsigned* count = sort_shared;                                            // [bins] of this block
  unsigned* base = count + bins;                                            // [bins] first place of a digit's slots here
  unsigned* all = base + bins;                                              // [warps][bins]
  unsigned* mine = all + warp * bins;
  const unsigned per = A.each / SORT_WARPS, begin = block * A.each + warp * per, turns = begin < A.S.rows ? min(per, A.S.rows - begin) : 0;
  const unsigned lower = (1u << lane) - 1;
  for (int pass = 0; pass < A.passes; pass++) {
    const int shift = pass * A.bits;
    unsigned key[CLUSTER_KEYS], row[CLUSTER_KEYS];
    bool slot[CLUSTER_KEYS];
#pragma unroll
    for (unsigned k = 0; k < CLUSTER_KEYS; k++) {
      row[k] = begin + k * 32 + lane;
      slot[k] = k * 32 + lane < turns;
    }
    if (pass == 0) {
      int t[CLUSTER_KEYS];
      slot_types(A.S, row, slot, t);
#pragma unroll
      for (unsigned k = 0; k < CLUSTER_KEYS; k++) key[k] = t[k] < 0 ? (unsigned)A.S.ntypes : (unsigned)t[k];  // empty slots come last
    } else {  // past the L1, which may hold what lay there before
#pragma unroll
      for (unsigned k = 0; k < CLUSTER_KEYS; k++) {
        key[k] = slot[k] ? __ldcg(A.key[(pass - 1) & 1] + row[k]) : 0;
        row[k] = slot[k] ? __ldcg(A.row[(pass - 1) & 1] + row[k]) : 0;
      }
    }
    for (unsigned b = lane; b < bins / 4; b += 32) reinterpret_cast<uint4*>(mine)[b] = make_uint4(0, 0, 0, 0);
    __syncwarp();
#pragma unroll
    for (unsigned k = 0; k < CLUSTER_KEYS; k++)
      if (slot[k]) atomicAdd(&mine[key[k] >> shift & mask], 1u);
    __syncthreads();
    for (unsigned b = tid; b < bins; b += SORT_THREADS) {
      unsigned at = 0;
#pragma unroll
      for (unsigned w0 = 0; w0 < SORT_WARPS; w0 += 16) {
        unsigned n[16];
#pragma unroll
        for (unsigned w = 0; w < 16; w++) n[w] = all[(w0 + w) * bins + b];
#pragma unroll
        for (unsigned w = 0; w < 16; w++) {
          all[(w0 + w) * bins + b] = at;
          at += n[w];
        }
      }
      count[b] = at;
    }
    cluster_arrive();
    cluster_wait();
    // digits' totals to their first places, a digit a thread
    unsigned sum = 0, off = 0;
    if (tid < bins) {
#pragma unroll
      for (unsigned c = 0; c < CLUSTER; c++) {
        const unsigned n = cluster_load(count + tid, c);
        sum += n;
        off += c < block ? n : 0;
      }
    }
    const bool last = pass == A.passes - 1;
    __syncthreads();
    if (last) cluster_arrive();  // the others' counts have been read: they may leave once all have come here
    unsigned run = sum;
    for (unsigned o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (lane == 31) warp_sum[warp] = run;
    __syncthreads();
    unsigned before = lane < warp ? warp_sum[lane] : 0;
    before = __reduce_add_sync(0xffffffffu, before);
    if (tid < bins) base[tid] = run - sum + before + off;
    __syncthreads();
    unsigned *key_out = A.key[pass & 1], *row_out = A.row[pass & 1];
#pragma unroll
    for (unsigned k = 0; k < CLUSTER_KEYS; k++) {
      if (k * 32 < turns) {
        const unsigned d = key[k] >> shift & mask, peers = same_digit(d, A.bits, slot[k]);
        const unsigned at = slot[k] ? base[d] + mine[d] + __popc(peers & lower) : ~0u;
        __syncwarp();
        if (slot[k] && (peers & lower) == 0) mine[d] += __popc(peers);
        __syncwarp();
        if (at < A.S.rows) {  // always, for types that nobody changes meanwhile
          key_out[at] = key[k];
          row_out[at] = row[k];
        }
      }
    }
    if (!last) cluster_arrive();  // this pass is written, and its counts have been read
    cluster_wait();
  }
}

size_t cluster_smem(int bits) { return (8 + 4 * SORT_WARPS) * ((size_t)1 << bits); }

size_t sort_smem(int bits) {
  const size_t bins = (size_t)1 << bits, slices = bins < SORT_THREADS ? SORT_THREADS / bins : 1;
  return 4 * bins + 8 * slices * bins + 2 * SORT_WARPS * bins;
}

// ---- sums of sorted slots ---------------------------------------------------------------------------------------------
struct PieceArgs {
  const unsigned *key, *row;
  unsigned n, ntypes, piece;
  int lanes;        // that share a piece, eight columns each; a power of two
  unsigned blocks;  // of PIECE_THREADS / lanes pieces
  int width;
  float* parts;     // [blocks][2][width]: of the type that comes in from the block before, of the one that goes on in the next
  float scale;
};

constexpr int PIECE_THREADS = 256, PIECE_SLOTS = 2048;  // slots of a block, at most

// The eight columns of a lane: next to each other where rows lie on 16 bytes, else every `lanes`th, so that neighbouring lanes touch
// neighbouring values (61 slots of 1402 types, 231 float32: 16 us with eight single values a lane next to each other).
template <bool VEC>
struct Columns {
  int first, step, width;
  __device__ __forceinline__ Columns(int tile, int lane, int lanes, int width_)
      : first(VEC ? (tile * lanes + lane) * 8 : tile * lanes * 8 + lane), step(VEC ? 1 : lanes), width(width_) {}
  __device__ __forceinline__ bool any() const { return first < width; }
  template <class T>
  __device__ __forceinline__ void store(T* row, const float (&v)[8]) const {
    if constexpr (VEC) {
      store_cols<T, 8, true>(row, first, width, v);
    } else {
#pragma unroll
      for (int c = 0; c < 8; c++)
        if (first + c * step < width) row[first + c * step] = from_float<T>(v[c]);
    }
  }
  __device__ __forceinline__ void load(const float* row, float (&v)[8]) const {  // of partial sums, which lie anywhere
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = first + c * step < width ? row[first + c * step] : 0.f;
  }
};
template <class T, bool VEC>
struct PieceRow {
  Raw<T, 8, true> raw;
  __device__ __forceinline__ void load(const T* row, const Columns<VEC>& C) { raw.load(row, C.first, C.width); }
  __device__ __forceinline__ float get(int c) const { return raw.get(c); }
};
template <class T>
struct PieceRow<T, false> {
  T v[8];
  __device__ __forceinline__ void load(const T* row, const Columns<false>& C) {
#pragma unroll
    for (int c = 0; c < 8; c++) v[c] = C.first + c * C.step < C.width ? row[C.first + c * C.step] : from_float<T>(0.f);
  }
  __device__ __forceinline__ float get(int c) const { return to_float(v[c]); }
};

// a block's sorted slots: key(1 .. here) and row(0 .. here - 1), key(0) and key(here + 1) those of the slots before and behind
struct TwoLists {
  const unsigned *keys, *rows;
  __device__ __forceinline__ unsigned key(unsigned i) const { return keys[i]; }
  __device__ __forceinline__ unsigned row(unsigned i) const { return rows[i]; }
};

// Sums of a block's sorted slots.  A group of lanes sums a piece type by type.  A type that crosses pieces is put together in shared memory by the
// group that it begins in; only what crosses blocks is left, in `parts` (46 us for 25000 slots, a tenth of them of one type,
// when every piece left its own).
template <class T, class O, bool VEC, bool DROP, class Sorted>
__device__ __forceinline__ void sum_pieces(const PieceArgs& A, const Sorted& sorted, float* heads, float* tails, unsigned here, int col_tile,
                                           const T* diff, long long diff_ld, O* grad, long long grad_ld, const Drop& D, float* parts) {
  constexpr int ROWS = VEC && sizeof(T) == 2 ? 8 : 4;  // whose loads are in flight together
  const int group = threadIdx.x / A.lanes, lane = threadIdx.x % A.lanes;
  const Columns<VEC> C(col_tile, lane, A.lanes, A.width);
  const unsigned begin = min(group * A.piece, here), end = min(begin + A.piece, here);
  const bool some = begin < end && C.any();
  const unsigned came = sorted.key(begin), goes = sorted.key(end + 1);
  float* head = heads + (size_t)group * A.lanes * 8 + lane * 8;
  float* tail = tails + (size_t)group * A.lanes * 8 + lane * 8;
  auto write = [&](unsigned type, float (&sum)[8]) {
#pragma unroll
    for (int c = 0; c < 8; c++) sum[c] *= A.scale;
    C.store(grad + (long long)type * grad_ld, sum);
  };
  if (some) {
    const DropKey K(D);
    // a group's lanes that are at work, and where in the warp it begins: they hand their bits round
    const int left = A.width - col_tile * A.lanes * 8, first_lane = (threadIdx.x & 31) - lane;
    const unsigned together = (left >= 32 ? ~0u : (1u << min(left, A.lanes)) - 1) >> (left >= 32 ? 32 - A.lanes : 0) << first_lane;
    float sum[8] = {};
    unsigned type = sorted.key(begin + 1);
    bool first = true;
    auto put = [&](bool last) {
      if (type >= A.ntypes) return;
      if (first && type == came) {
#pragma unroll
        for (int c = 0; c < 8; c++) head[c] = sum[c];
      } else if (last && type == goes) {
#pragma unroll
        for (int c = 0; c < 8; c++) tail[c] = sum[c];
      } else {
        write(type, sum);
      }
    };
    for (unsigned i = begin; i < end; i += ROWS) {
      PieceRow<T, VEC> v[ROWS];
#pragma unroll
      for (int j = 0; j < ROWS; j++)
        if (i + j < end && sorted.key(i + j + 1) < A.ntypes) v[j].load(diff + (long long)sorted.row(i + j) * diff_ld, C);
#pragma unroll
      for (int j = 0; j < ROWS; j++) {
        if (i + j >= end) break;
        const unsigned t = sorted.key(i + j + 1);
        if (t != type) {
          put(false);
          first = false;
          type = t;
#pragma unroll
          for (int c = 0; c < 8; c++) sum[c] = 0.f;
        }
        if (type >= A.ntypes) continue;
        if (DROP) {
          const unsigned bits = kept8(D, K, sorted.row(i + j), col_tile * A.lanes + lane);
#pragma unroll
          for (int c = 0; c < 8; c++) {
            const int at = lane + c * A.lanes;  // of the tile's columns
            const bool stays = VEC ? bits >> c & 1 : __shfl_sync(together, bits, first_lane + at / 8) >> (at & 7) & 1;
            sum[c] += stays ? v[j].get(c) * D.scale : 0.f;
          }
        } else {
#pragma unroll
          for (int c = 0; c < 8; c++) sum[c] += v[j].get(c);
        }
      }
    }
    put(true);
  }
  __syncthreads();
  if (!some) return;
  // The heads of pieces from `p` on, while the type goes on; true: beyond the block.  Which piece is the first that does not begin with the
  // type is found by halves (a key and a head after the other: 15.6 us instead of 13.9 for 25551 slots of 350 types, 13.2 instead of 9.9
  // for 1024 of five and 1000 columns).
  const unsigned pieces = (here + A.piece - 1) / A.piece;
  auto follow = [&](unsigned type, unsigned p, float (&sum)[8]) {
    unsigned least = p, most = pieces;
    while (least < most) {
      const unsigned half = (least + most) / 2;
      if (sorted.key(half * A.piece + 1) == type) least = half + 1;
      else most = half;
    }
#pragma unroll 4
    for (; p < least; p++) {
      const float* h = heads + (size_t)p * A.lanes * 8 + lane * 8;
#pragma unroll
      for (int c = 0; c < 8; c++) sum[c] += h[c];
    }
    return least == pieces && sorted.key(here) == type && sorted.key(here + 1) == type;
  };
  auto put_part = [&](float* to, const float (&sum)[8]) {
#pragma unroll
    for (int c = 0; c < 8; c++)
      if (C.first + c * C.step < A.width) to[C.first + c * C.step] = sum[c];
  };
  const unsigned t0 = sorted.key(begin + 1), t1 = sorted.key(end);
  if (group == 0 && t0 == came && t0 < A.ntypes) {
    float sum[8] = {};
    follow(t0, 0, sum);
    put_part(parts, sum);
  }
  if (goes == t1 && t1 < A.ntypes && !(t0 == t1 && came == t0)) {
    float sum[8];
#pragma unroll
    for (int c = 0; c < 8; c++) sum[c] = tail[c];
    if (follow(t1, group + 1, sum)) put_part(parts + A.width, sum);
    else write(t1, sum);
  }
}

template <class T, class O, bool VEC, bool DROP>
__global__ void __launch_bounds__(PIECE_THREADS, DROP ? 2 : 3) k_type_pieces(PieceArgs A, const T* diff, long long diff_ld, O* grad, long long grad_ld, Drop D) {
  __shared__ unsigned keys[PIECE_SLOTS + 2], rows[PIECE_SLOTS];
  __shared__ float heads[PIECE_THREADS * 8], tails[PIECE_THREADS * 8];
  wait_for_stream();
  const unsigned slots = PIECE_THREADS / A.lanes * A.piece, first_slot = blockIdx.x * slots, here = min(slots, A.n - first_slot);
  for (unsigned i = threadIdx.x; i < here + 2; i += PIECE_THREADS) {
    const unsigned at = first_slot + i;  // keys[i] is that of the slot before
    keys[i] = at > 0 && at <= A.n ? A.key[at - 1] : ~0u;
    if (i < here) rows[i] = A.row[at];
  }
  __syncthreads();
  sum_pieces<T, O, VEC, DROP>(A, TwoLists{keys, rows}, heads, tails, here, blockIdx.y, diff, diff_ld, grad, grad_ld, D,
                                             A.parts + (size_t)blockIdx.x * 2 * A.width);
}

// ---- up to 1024 slots, in one launch ---------------------------------------------------------------------------------------
// The first blocks sort all slots in shared memory, (type, slot) as one word each, by bitonic merges (Batcher, "Sorting networks and their
// applications", 1968), and sum them for 8 * lanes columns each; the others clear the rows of the types that no
// slot has.  (Three launches otherwise: 1000 slots of 5000 types 16 us, 300 of 100000 types 14 us.)
constexpr int SMALL_THREADS = 512, SMALL_SLOTS = 1024, SMALL_RANGE = 32768;  // types whose rows a block clears, at most
constexpr int SMALL_TYPES = 1 << 21;

template <class T, class O, bool VEC, bool DROP>
__global__ void __launch_bounds__(SMALL_THREADS) k_type_small(Slots S, PieceArgs A, unsigned sum_blocks, unsigned range, FastDiv by_units, const T* diff,
                                                              long long diff_ld, O* grad, long long grad_ld, Drop D) {
  __shared__ unsigned keys[SMALL_SLOTS + 2], rows[SMALL_SLOTS];
  __shared__ float heads[SMALL_THREADS * 8], tails[SMALL_THREADS * 8];
  const unsigned tid = threadIdx.x;
  wait_for_stream();
  const unsigned slot[2] = {tid, tid + SMALL_THREADS};
  const bool in[2] = {slot[0] < A.n, slot[1] < A.n};
  if (blockIdx.x >= sum_blocks) {
    const unsigned first = (blockIdx.x - sum_blocks) * range, types = min(range, A.ntypes - first);
    unsigned* met = reinterpret_cast<unsigned*>(heads);  // a bit a type
    for (unsigned i = tid; i < (types + 31) / 32; i += SMALL_THREADS) met[i] = 0;
    __syncthreads();
    int t[2];
    slot_types(S, slot, in, t);
    for (int k = 0; k < 2; k++)
      if (in[k] && t[k] >= 0 && (unsigned)t[k] - first < types) atomicOr(&met[((unsigned)t[k] - first) / 32], 1u << (((unsigned)t[k] - first) & 31));
    __syncthreads();
    // eight values a thread and turn where rows lie on 16 bytes, else one, by columns
    const unsigned units = by_units.d;
    for (unsigned i = tid; i < types * units; i += SMALL_THREADS) {
      const unsigned type = by_units(i), at = i - type * units;
      if (met[type / 32] >> (type & 31) & 1) continue;
      O* row = grad + (long long)(first + type) * grad_ld;
      if constexpr (VEC) {
        const float zeros[8] = {};
        store_cols<O, 8, true>(row, (int)at * 8, A.width, zeros);
      } else {
        row[at] = from_float<O>(0.f);
      }
    }
    return;
  }
  unsigned n2 = 64;  // slots that the network sorts
  while (n2 < A.n) n2 *= 2;
  {
    int t[2];
    slot_types(S, slot, in, t);
    for (int k = 0; k < 2; k++)
      if (slot[k] < n2) rows[slot[k]] = in[k] ? (t[k] < 0 ? A.ntypes : (unsigned)t[k]) << 10 | slot[k] : ~0u;  // empty slots come last
  }
  __syncthreads();
  for (unsigned size = 2; size <= n2; size *= 2)
    for (unsigned stride = size / 2; stride; stride /= 2) {
      // a warp's pairs lie in its own 64 words where they are up to 32 apart: others' are waited for at 64 and more, and behind them
      if (stride >= 32) __syncthreads();
      else __syncwarp();
      if (tid < n2 / 2) {
        const unsigned i = 2 * tid - (tid & (stride - 1)), a = rows[i], b = rows[i + stride];
        if ((a > b) == ((i & size) == 0)) {
          rows[i] = b;
          rows[i + stride] = a;
        }
      }
    }
  __syncthreads();
  unsigned word[2];
  for (int k = 0; k < 2; k++) word[k] = in[k] ? rows[slot[k]] : 0;
  __syncthreads();
  for (int k = 0; k < 2; k++)
    if (in[k]) {
      keys[slot[k] + 1] = word[k] >> 10;
      rows[slot[k]] = word[k] & 1023;
    }
  if (tid == 0) keys[0] = keys[A.n + 1] = ~0u;
  __syncthreads();
  sum_pieces<T, O, VEC, DROP>(A, TwoLists{keys, rows}, heads, tails, A.n, blockIdx.x, diff, diff_ld, grad, grad_ld, D, nullptr);
}

// ---- some hundred types, in one launch -------------------------------------------------------------------------------------
// A cluster has every fifteenth type (types are often numbered by how common they are), a block of it an eighth of the slots: it finds
// those of its types, in order, sorts them in shared memory, (type, slot) as one word each, and sums them to a table there; the blocks'
// tables are added up at the end.  (A block alone for a share of the types waits for the one that many slots have: 25551 slots of
// 350 types, one in eight of one, 37.8 us.)
constexpr int RANGE_THREADS = 512, RANGE_WARPS = RANGE_THREADS / 32, RANGE_TYPES = 64;
constexpr unsigned RANGES = 15;  // clusters that fit at once: 16 take 16.6 us for those slots, 15 13.9

__host__ __device__ constexpr unsigned range_share(unsigned rows) {  // slots of a warp
  return (rows + CLUSTER * RANGE_THREADS - 1) / (CLUSTER * RANGE_THREADS) * 32;
}
// shared memory: a block's words, then its lists, a slot and a type for each, whose place the partial sums take in the end, then the table and counts
__host__ __device__ constexpr size_t range_words(unsigned rows) { return ((size_t)range_share(rows) * RANGE_WARPS + 2 + 3) / 4 * 16; }
__host__ __device__ constexpr size_t range_lists(unsigned rows) {
  const size_t lists = (size_t)range_share(rows) * RANGE_WARPS * 3, sums = RANGE_THREADS * 8 * 2 * 4;
  return lists > sums ? lists : sums;
}
size_t range_smem(unsigned rows, unsigned types, int lanes) {
  return range_words(rows) + range_lists(rows) + (size_t)types * lanes * 32 + RANGE_WARPS * RANGE_TYPES * 4;
}

struct OneList {
  const unsigned* words;
  unsigned first;  // slot of the block
  __device__ __forceinline__ unsigned key(unsigned i) const { return words[i] >> 16; }
  __device__ __forceinline__ unsigned row(unsigned i) const { return first + (words[i + 1] & 0xffffu); }
};

template <class T, class O, bool VEC, bool DROP>
__global__ void __launch_bounds__(RANGE_THREADS) k_type_ranges(Slots S, PieceArgs A, FastDiv by_ranges, const T* diff, long long diff_ld,
                                                               O* grad, long long grad_ld, Drop D) {
  extern __shared__ float4 range_shared[];
  __shared__ unsigned total;
  char* shared = reinterpret_cast<char*>(range_shared);
  const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid / 32, lower = (1u << lane) - 1, share = range_share(S.rows);
  const unsigned rank = blockIdx.x % CLUSTER, range = blockIdx.x / CLUSTER, ranges = by_ranges.d, here_types = (A.ntypes - range + ranges - 1) / ranges;
  unsigned* words = reinterpret_cast<unsigned*>(shared);
  unsigned short* slots = reinterpret_cast<unsigned short*>(shared + range_words(S.rows)) + warp * share;
  unsigned char* types = reinterpret_cast<unsigned char*>(shared + range_words(S.rows)) + 2 * RANGE_WARPS * share + warp * share;
  float* heads = reinterpret_cast<float*>(shared + range_words(S.rows));
  float* table = reinterpret_cast<float*>(shared + range_words(S.rows) + range_lists(S.rows));
  const unsigned cols = A.lanes * 8;
  unsigned (*count)[RANGE_TYPES] = reinterpret_cast<unsigned (*)[RANGE_TYPES]>(table + here_types * cols);  // of each warp and type
  for (unsigned i = tid; i < here_types * cols / 4; i += RANGE_THREADS) reinterpret_cast<float4*>(table)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = tid; i < RANGE_WARPS * RANGE_TYPES; i += RANGE_THREADS) count[i / RANGE_TYPES][i % RANGE_TYPES] = 0;
  __syncthreads();
  wait_for_stream();
  const unsigned block_first = rank * share * RANGE_WARPS, begin = block_first + warp * share, end = min(begin + share, S.rows);
  unsigned found = 0;
  constexpr int N = 8;  // that are looked up together
  for (unsigned i0 = begin; i0 < end; i0 += 32 * N) {
    unsigned row[N];
    bool in[N];
    int t[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
      row[k] = i0 + k * 32 + lane;
      in[k] = row[k] < end;
    }
    slot_types(S, row, in, t);
#pragma unroll
    for (int k = 0; k < N; k++) {
      const unsigned type = by_ranges(t[k] < 0 ? 0 : (unsigned)t[k]);
      const bool mine = t[k] >= 0 && (unsigned)t[k] - type * ranges == range;
      const unsigned all = __ballot_sync(0xffffffffu, mine);
      if (mine) {
        const unsigned at = found + __popc(all & lower);
        slots[at] = (unsigned short)(row[k] - block_first);
        types[at] = (unsigned char)type;
        atomicAdd(&count[warp][type], 1u);
      }
      found += __popc(all);
    }
  }
  __syncthreads();
  if (warp == 0) {  // a lane has two types: where each warp's slots of them go
    unsigned n[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < RANGE_WARPS; w++) {
      n[0] += count[w][2 * lane];
      n[1] += count[w][2 * lane + 1];
    }
    unsigned run = n[0] + n[1];
    for (unsigned o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (lane == 31) total = run;
    unsigned at[2] = {run - n[0] - n[1], run - n[1]};
#pragma unroll
    for (int w = 0; w < RANGE_WARPS; w++) {
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const unsigned m = count[w][2 * lane + k];
        count[w][2 * lane + k] = at[k];
        at[k] += m;
      }
    }
  }
  __syncthreads();
  const unsigned here = total;
  for (unsigned i0 = 0; i0 < found; i0 += 32) {
    const bool slot = i0 + lane < found;
    const unsigned type = slot ? types[i0 + lane] : 0, peers = same_digit(type, 6, slot);
    if (slot) words[1 + count[warp][type] + __popc(peers & lower)] = type << 16 | slots[i0 + lane];
    __syncwarp();
    if (slot && (peers & lower) == 0) count[warp][type] += __popc(peers);
    __syncwarp();
  }
  if (tid == 0) words[0] = words[here + 1] = ~0u;
  __syncthreads();
  PieceArgs P = A;
  const unsigned groups = RANGE_THREADS / A.lanes;
  P.ntypes = here_types;
  P.piece = max(4u, (here + groups - 1) / groups);  // four slots are one round of loads
  P.scale = 1.f;
  sum_pieces<T, float, VEC, DROP>(P, OneList{words, block_first}, heads, heads + RANGE_THREADS * 8, here, 0, diff, diff_ld, table, (long long)cols, D, nullptr);
  cluster_arrive();
  cluster_wait();
  for (unsigned i = rank * RANGE_THREADS + tid; i < here_types * cols; i += CLUSTER * RANGE_THREADS) {
    const unsigned type = i / cols, col = i % cols;
    float part[CLUSTER], sum = 0.f;
#pragma unroll
    for (unsigned c = 0; c < CLUSTER; c++) part[c] = __uint_as_float(cluster_load(reinterpret_cast<const unsigned*>(table) + i, c));
#pragma unroll
    for (unsigned c = 0; c < CLUSTER; c++) sum += part[c];
    if ((int)col < A.width) grad[(long long)(type * ranges + range) * grad_ld + col] = from_float<O>(sum * A.scale);
  }
  cluster_arrive();  // the others read what lies here
  cluster_wait();
}

// a type that begins in a block and goes on: its parts, block after block
template <class O, bool VEC>
__global__ void __launch_bounds__(PIECE_THREADS) k_type_joins(PieceArgs A, O* grad, long long grad_ld) {
  wait_for_stream();
  const unsigned at = blockIdx.x * PIECE_THREADS + threadIdx.x, block = at / A.lanes, slots = PIECE_THREADS / A.lanes * A.piece;
  const Columns<VEC> C(blockIdx.y, at % A.lanes, A.lanes, A.width);
  if (block + 1 >= A.blocks || !C.any()) return;
  // all that a type which ends in the next block needs is on its way before it is known whether there is one
  const unsigned begin = block * slots, end = begin + slots, type = A.key[end - 1], goes = A.key[end], came = begin > 0 ? A.key[begin - 1] : ~0u;
  const unsigned after = block + 2 < A.blocks ? A.key[end + slots] : ~0u;
  float sum[8], more[8];
  C.load(A.parts + ((size_t)block * 2 + 1) * A.width, sum);
  C.load(A.parts + ((size_t)block + 1) * 2 * A.width, more);
  if (type >= A.ntypes || goes != type || came == type) return;
#pragma unroll
  for (int c = 0; c < 8; c++) sum[c] += more[c];
  unsigned p = after == type ? block + 2 : A.blocks;
  while (p + 4 <= A.blocks && A.key[(p + 3) * slots] == type) {
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; j++) C.load(A.parts + (size_t)(p + j) * 2 * A.width, v[j]);
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int c = 0; c < 8; c++) sum[c] += v[j][c];
    p += 4;
  }
  for (; p < A.blocks && A.key[p * slots] == type; p++) {
    C.load(A.parts + (size_t)p * 2 * A.width, more);
#pragma unroll
    for (int c = 0; c < 8; c++) sum[c] += more[c];
  }
#pragma unroll
  for (int c = 0; c < 8; c++) sum[c] *= A.scale;
  C.store(grad + (long long)type * grad_ld, sum);
}

// ---- the plan: a function of the sizes alone, so that the workspace and the call agree ----------------------------------------
struct Plan {
  bool tables, small, ranges;
  // few types
  unsigned blocks, per;
  int warps;
  size_t table_smem;
  // sorted
  unsigned tiles, tile;  // tiles 0: one cluster sorts, `tile` slots a block
  int passes, bits;
  unsigned piece, piece_blocks;
  int lanes;
  size_t key[2], row[2], counts, parts, bytes;
};

constexpr size_t TABLE_SMEM = SMEM_MOST;  // an SM's
constexpr int TABLE_WARPS_LEAST = 4, TABLE_WARPS_MOST = 16;
// Tiles of 32 columns, and slots times tiles, up to which tables are kept: 200000 slots of 28 types and 128 float32 take 45.5 us with them
// and 46.5 sorted, of 256 bfloat16 78 and 64, 20000 of 200 float32 10.6 and 23.5.  Set by four tiles: of one tile (28 columns) tables take 36.8 for
// 1048576 slots, and one slot more, sorted, 73.
constexpr unsigned TABLE_TILES = 8, TABLE_WORK = 1 << 20;

// Slots times columns, and columns, up to which clusters share the types.  In us, shared and sorted: 25551 slots of 350 types and 45 float16
// 13.6 and 18.4, 10000 of 300 and 8 float32 6.9 and 17, 60000 of 400 and 128 bfloat16 20 and 26, 20000 of 1900 and 64 float32 15 and 20; 30000 of 300
// and 1000 float16 55 and 38, 1500 of 120 and 300 float32 13.2 and 12.5.  Where one type has all slots, which the sizes do not tell, eight blocks
// do all: the first 46 and 30, without dropout 27 and 29, the third 72 and 51.
constexpr size_t RANGE_WORK = 1 << 23, RANGE_SMEM = 200 << 10;

Plan plan_for(unsigned rows, int V, int width) {
  Plan p = {};
  if (V == 0 || width == 0 || rows == 0) {
    p.bytes = STATUS_FRONT;
    return p;
  }
  // tables: four a warp; fewer than four warps an SM have too few loads in flight
  const size_t warp_smem = (size_t)4 * V * TABLE_COLS * 4;
  const unsigned col_tiles = ((unsigned)width + TABLE_COLS - 1) / TABLE_COLS;
  if (warp_smem * TABLE_WARPS_LEAST <= TABLE_SMEM && col_tiles <= TABLE_TILES && (size_t)rows * col_tiles <= TABLE_WORK) {
    p.warps = (int)(TABLE_SMEM / warp_smem < TABLE_WARPS_MOST ? TABLE_SMEM / warp_smem : TABLE_WARPS_MOST);
    const unsigned all = (rows + 31) / 32;  // warps that find 32 slots
    if (all < 148u * p.warps) p.warps = all / 148 < TABLE_WARPS_LEAST ? TABLE_WARPS_LEAST : (int)(all / 148);
    p.blocks = (all + p.warps - 1) / p.warps < 148 ? (all + p.warps - 1) / p.warps : 148;
    // the blocks' tables are written and read once more: worth it while they are a fraction of the gradients
    if ((size_t)p.blocks * V <= rows || p.blocks == 1) {
      p.tables = true;
      p.table_smem = warp_smem * p.warps;
      const unsigned warps = p.blocks * p.warps;
      p.per = ((rows + warps - 1) / warps + 31) / 32 * 32;
      p.blocks = (unsigned)(((unsigned long long)rows + (unsigned long long)p.per * p.warps - 1) / ((unsigned long long)p.per * p.warps));
      p.bytes = STATUS_FRONT + (size_t)p.blocks * V * width * 4;
      return p;
    }
  }
  if (rows <= SMALL_SLOTS && V < SMALL_TYPES && width <= 1 << 20) {
    p.small = true;
    // as many lanes as leave pieces of four slots (one round of loads), more where the blocks, which all sort, would be more than SMs
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes * 8 < width && (rows * p.lanes * 2 <= 4 * SMALL_THREADS || width > 148 * 8 * p.lanes)) p.lanes *= 2;
    const unsigned groups = SMALL_THREADS / p.lanes;
    p.piece = (rows + groups - 1) / groups;
    // blocks that clear: about 512 groups of eight columns each, and a bit a type
    const unsigned long long eights = (unsigned long long)V * ((width + 7) / 8);
    unsigned blocks = (unsigned)(eights / 512 + 1 < 592 ? eights / 512 + 1 : 592);
    if (blocks < ((unsigned)V + SMALL_RANGE - 1) / SMALL_RANGE) blocks = ((unsigned)V + SMALL_RANGE - 1) / SMALL_RANGE;
    p.per = (V + blocks - 1) / blocks;  // types of a block
    p.blocks = (V + p.per - 1) / p.per;
    p.bytes = STATUS_FRONT;
    return p;
  }
  if (V <= (int)(2 * RANGES * RANGE_TYPES) && width <= 256 && (size_t)rows * width <= RANGE_WORK) {
    p.lanes = 1;
    while (p.lanes < 32 && p.lanes * 8 < width) p.lanes *= 2;
    unsigned ranges = ((unsigned)V + RANGE_TYPES - 1) / RANGE_TYPES;
    if (ranges < RANGES) ranges = RANGES;
    p.per = (V + ranges - 1) / ranges;
    p.blocks = ranges < (unsigned)V ? ranges : V;
    if (range_smem(rows, p.per, p.lanes) <= RANGE_SMEM) {
      p.ranges = true;
      p.bytes = STATUS_FRONT;
      return p;
    }
  }
  int key_bits = 2, most = 2;  // two bits a pass at least, with more than 2^30 slots too: 31 bits take 16 passes
  while (key_bits < 31 && (unsigned)V >> key_bits) key_bits++;
  if (rows <= CLUSTER * CLUSTER_KEYS * SORT_THREADS) {
    p.tile = (rows + CLUSTER * SORT_THREADS - 1) / (CLUSTER * SORT_THREADS) * SORT_THREADS;
    most = CLUSTER_BITS_MOST;
  } else {
    p.tile = SORT_THREADS;
    while ((rows + p.tile - 1) / p.tile > 148 && p.tile < SORT_TILE_MOST) p.tile += SORT_THREADS;
    p.tiles = (rows + p.tile - 1) / p.tile;
    // a block reads all tiles' counts: half a megabyte at most
    while (most < SORT_BITS_MOST && ((size_t)p.tiles << (most + 1)) <= 1 << 17) most++;
  }
  p.passes = (key_bits + most - 1) / most;
  p.bits = (key_bits + p.passes - 1) / p.passes;
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes * 8 < width) p.lanes *= 2;
  const unsigned cols = (width + p.lanes * 8 - 1) / (p.lanes * 8);
  // pieces for 16 warps an SM, of 4 to 32 slots: for 64, 16384 slots of 1024 bfloat16 take 46 us instead of 42
  const size_t want = (size_t)rows * cols * p.lanes / (148 * 16 * 32);
  p.piece = 4;
  while (p.piece < 32 && p.piece < want && p.piece * 2 * (PIECE_THREADS / p.lanes) <= PIECE_SLOTS) p.piece *= 2;
  const unsigned slots = p.piece * (PIECE_THREADS / p.lanes);
  p.piece_blocks = (rows + slots - 1) / slots;
  size_t at = STATUS_FRONT;
  for (int k = 0; k < 2; k++) {
    p.key[k] = at;
    at += aligned256((size_t)rows * 4);
    p.row[k] = at;
    at += aligned256((size_t)rows * 4);
  }
  p.counts = at;
  at += aligned256(((size_t)p.tiles << p.bits) * 4);
  p.parts = at;
  at += (size_t)p.piece_blocks * 2 * width * 4;
  p.bytes = at;
  return p;
}

template <class T, class O>
cudaError_t by_tables(const Slots& S, const Plan& p, const lmg_vectors* diff, const lmg_vectors* grad, int width, float scale, const Drop& D,
                      char* ws, long* launches, cudaStream_t st) {
  float* parts = reinterpret_cast<float*>(ws + STATUS_FRONT);
  O* g = static_cast<O*>(grad->data);
  const bool vec = rows_aligned(diff);
  const auto kernel = vec ? (drops(D) ? k_type_tables<T, O, true, true> : k_type_tables<T, O, true, false>)
                          : (drops(D) ? k_type_tables<T, O, false, true> : k_type_tables<T, O, false, false>);
  cudaError_t e = allow_smem(kernel, p.table_smem);
  if (e == cudaSuccess)
    e = launch_early(kernel, dim3(p.blocks, (width + TABLE_COLS - 1) / TABLE_COLS), 32 * p.warps, p.table_smem, st, S, p.per,
                     static_cast<const T*>(diff->data), diff->ld, width, parts, g, grad->ld, scale, D);
  if (e != cudaSuccess) return e;
  ++*launches;
  if (p.blocks == 1) return e;
  ++*launches;
  return launch_early(k_table_sums<O>, dim3((unsigned)(((size_t)S.ntypes * width + 31) / 32)), 1024, 0, st, parts, (int)p.blocks, S.ntypes, width, g,
                      grad->ld, scale);
}

template <class T, class O>
cudaError_t by_network(const Slots& S, const Plan& p, const lmg_vectors* diff, const lmg_vectors* grad, int width, float scale, const Drop& D,
                       char*, long* launches, cudaStream_t st) {
  PieceArgs P = {};
  P.n = S.rows;
  P.ntypes = (unsigned)S.ntypes;
  P.piece = p.piece;
  P.lanes = p.lanes;
  P.width = width;
  P.scale = scale;
  const bool vec = rows_aligned(diff) && rows_aligned(grad);
  const auto kernel = vec ? (drops(D) ? k_type_small<T, O, true, true> : k_type_small<T, O, true, false>)
                          : (drops(D) ? k_type_small<T, O, false, true> : k_type_small<T, O, false, false>);
  const unsigned sums = (width + p.lanes * 8 - 1) / (p.lanes * 8);
  ++*launches;
  return launch_early(kernel, dim3(sums + p.blocks), SMALL_THREADS, 0, st, S, P, sums, p.per, FastDiv(vec ? (unsigned)(width + 7) / 8 : (unsigned)width),
                      static_cast<const T*>(diff->data), diff->ld, static_cast<O*>(grad->data), grad->ld, D);
}

template <class T, class O>
cudaError_t by_ranges(const Slots& S, const Plan& p, const lmg_vectors* diff, const lmg_vectors* grad, int width, float scale, const Drop& D,
                      char*, long* launches, cudaStream_t st) {
  PieceArgs P = {};
  P.n = S.rows;
  P.ntypes = (unsigned)S.ntypes;
  P.lanes = p.lanes;
  P.width = width;
  P.scale = scale;
  const bool vec = rows_aligned(diff);
  const auto kernel = vec ? (drops(D) ? k_type_ranges<T, O, true, true> : k_type_ranges<T, O, true, false>)
                          : (drops(D) ? k_type_ranges<T, O, false, true> : k_type_ranges<T, O, false, false>);
  const size_t smem = range_smem(S.rows, p.per, p.lanes);
  const cudaError_t e = allow_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  ++*launches;
  return launch_clusters(kernel, p.blocks * CLUSTER, CLUSTER, RANGE_THREADS, smem, st, S, P, FastDiv(p.blocks), static_cast<const T*>(diff->data),
                         diff->ld, static_cast<O*>(grad->data), grad->ld, D);
}

template <class T, class O>
cudaError_t by_sort(const Slots& S, const Plan& p, const lmg_vectors* diff, const lmg_vectors* grad, int width, float scale, const Drop& D,
                    char* ws, long* launches, cudaStream_t st) {
  // the table's gradient is cleared meanwhile, in shares of the sort's launches; where rows have gaps, or begin off 16 bytes, before
  const size_t size = sizeof(O), total = (size_t)S.ntypes * width * size;
  char* g = static_cast<char*>(grad->data);
  cudaError_t e = cudaSuccess;
  const bool dense = grad->ld == width && reinterpret_cast<uintptr_t>(g) % 16 == 0;
  if (!dense) e = cudaMemset2DAsync(g, grad->ld * size, 0, width * size, S.ntypes, st);
  if (e != cudaSuccess) return e;
  const int parts = p.tiles ? 2 * p.passes : 1;
  const size_t clears = dense ? total : 0, share = (clears / 16 + parts) / parts * 16;
  auto clear = [&](int k, Clear& c) {
    const size_t from = share * k < clears ? share * k : clears;
    c.p = g + from;
    c.bytes = clears - from < share ? clears - from : share;
    const size_t blocks = (c.bytes / 16 + SORT_THREADS * 4) / (SORT_THREADS * 4);
    return c.bytes == 0 ? 0u : (unsigned)(blocks < 296 ? blocks : 296);
  };
  unsigned *key[2], *row[2];
  for (int k = 0; k < 2; k++) {
    key[k] = reinterpret_cast<unsigned*>(ws + p.key[k]);
    row[k] = reinterpret_cast<unsigned*>(ws + p.row[k]);
  }
  if (p.tiles == 0) {
    ClusterSortArgs A = {S, p.tile, p.passes, p.bits, {key[0], key[1]}, {row[0], row[1]}, {}};
    const unsigned blocks = clear(0, A.clear);
    const size_t smem = cluster_smem(p.bits);
    if ((e = allow_smem(k_sort_cluster, smem)) != cudaSuccess) return e;
    e = launch_clusters(k_sort_cluster, CLUSTER + (blocks + CLUSTER - 1) / CLUSTER * CLUSTER, CLUSTER, SORT_THREADS, smem, st, A);
    if (e != cudaSuccess) return e;
    ++*launches;
  } else {
    SortArgs A = {};
    A.S = S;
    A.tiles = p.tiles;
    A.tile = p.tile;
    A.bits = p.bits;
    A.counts = reinterpret_cast<unsigned*>(ws + p.counts);
    const size_t smem = sort_smem(p.bits);
    if ((e = allow_smem(k_sort_move, smem)) != cudaSuccess) return e;
    for (int k = 0; k < p.passes; k++) {
      A.shift = k * p.bits;
      A.key_in = k ? key[(k - 1) & 1] : nullptr;
      A.row_in = k ? row[(k - 1) & 1] : nullptr;
      A.key_out = key[k & 1];
      A.row_out = row[k & 1];
      unsigned blocks = p.tiles + clear(2 * k, A.clear);
      if ((e = launch_early(k_sort_count, dim3(blocks), SORT_THREADS, 0, st, A)) != cudaSuccess) return e;
      blocks = p.tiles + clear(2 * k + 1, A.clear);
      if ((e = launch_early(k_sort_move, dim3(blocks), SORT_THREADS, smem, st, A)) != cudaSuccess) return e;
      *launches += 2;
    }
  }
  PieceArgs P = {};
  P.key = key[(p.passes - 1) & 1];
  P.row = row[(p.passes - 1) & 1];
  P.n = S.rows;
  P.ntypes = (unsigned)S.ntypes;
  P.piece = p.piece;
  P.blocks = p.piece_blocks;
  P.lanes = p.lanes;
  P.width = width;
  P.parts = reinterpret_cast<float*>(ws + p.parts);
  P.scale = scale;
  const bool vec = rows_aligned(diff) && rows_aligned(grad);
  const unsigned cols = (width + p.lanes * 8 - 1) / (p.lanes * 8);
  const auto pieces = vec ? (drops(D) ? k_type_pieces<T, O, true, true> : k_type_pieces<T, O, true, false>)
                          : (drops(D) ? k_type_pieces<T, O, false, true> : k_type_pieces<T, O, false, false>);
  e = launch_early(pieces, dim3(p.piece_blocks, cols), PIECE_THREADS, 0, st, P, static_cast<const T*>(diff->data), diff->ld, static_cast<O*>(grad->data), grad->ld, D);
  if (e != cudaSuccess) return e;
  ++*launches;
  if (p.piece_blocks == 1) return e;
  ++*launches;
  const dim3 grid((unsigned)(((size_t)p.piece_blocks * p.lanes + PIECE_THREADS - 1) / PIECE_THREADS), cols);
  return launch_early(vec ? k_type_joins<O, true> : k_type_joins<O, false>, grid, PIECE_THREADS, 0, st, P, static_cast<O*>(grad->data), grad->ld);
}

}  // namespace
}  // namespace lmg

extern "C" {

int lmg_embed_types_backward(const lmg_slots* slots, int ntypes, int width, const lmg_vectors* diff, float scale,
                             const lmg_dropout_spec* drop, const lmg_vectors* table_gradients, void* workspace,
                             size_t workspace_bytes, void* stream) {
  using namespace lmg;
  int rc;
  if ((rc = check_slots(slots, width)) || (rc = check_index(slots, ntypes)) || (rc = check_drop(drop))) return rc;
  if (width > 1 << 23) return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "table gradients of more than 2^23 columns");
  if (ntypes == 0 || width == 0) return LMG_OK;
  if ((rc = check_vectors(table_gradients, width, "table gradients"))) return rc;
  const bool none = slots->batch == 0 || slots->max_atoms == 0;
  if (!none && (rc = check_vectors(diff, width, "diff"))) return rc;
  if (!none && diff->type != table_gradients->type && table_gradients->type != LMG_FLOAT32)
    return vectors_fail(LMG_ERR_INVALID_ARGUMENT, "diff and table gradients differ in type, and the gradients are not float32");
  const Slots S = to_slots(slots, ntypes);
  const Plan p = plan_for(S.rows, ntypes, width);
  if (workspace == nullptr || workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return vectors_fail(LMG_ERR_WORKSPACE, "workspace too small for the gradient of a table, or off 16 bytes");
  const cudaStream_t st = (cudaStream_t)stream;
  if (none) {
    const size_t size = element_bytes(table_gradients->type);
    const cudaError_t e = cudaMemset2DAsync(table_gradients->data, table_gradients->ld * size, 0, width * size, ntypes, st);
    return e == cudaSuccess ? LMG_OK : vectors_cuda(e, "gradient of a table");
  }
  const Drop D = to_drop(drop);
  long launches = 0;
  const cudaError_t e = by_vector_types<false, true>(diff->type, table_gradients->type, [&](auto t, auto o) {
    const auto by = p.tables ? by_tables<decltype(t), decltype(o)> : p.small ? by_network<decltype(t), decltype(o)>
                    : p.ranges ? by_ranges<decltype(t), decltype(o)> : by_sort<decltype(t), decltype(o)>;
    return by(S, p, diff, table_gradients, width, scale, D, static_cast<char*>(workspace), &launches, st);
  });
  lmg_internal_count_launches(launches);
  return e == cudaSuccess ? LMG_OK : vectors_cuda(e, "gradient of a table");
}

}  // extern "C"

namespace lmg {
size_t embed_backward_bytes(unsigned rows, int ntypes, int width) { return plan_for(rows, ntypes, width).bytes; }
}  // namespace lmg

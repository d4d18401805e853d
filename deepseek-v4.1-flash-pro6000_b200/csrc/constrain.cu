// Constraints on logits rows: token penalties, a bias list per sequence and the grammar bitmask, out of place or in place
// (include/ds41_b200.h has the rule).  A row is a stream: every logit that the mask allows is read once and every one written once,
// so what bounds large batches is the memory; a single row is bounded by the history's way through the counters.
//
// One team of up to eight CTAs per row, each with a slice of at most 16384 ids: their occurrences fit 16-bit counters in 32 KB of
// shared memory, counted with shared-memory atomics.  Every CTA reads the whole history (from L2 after the first of them).
// Counters and mask bits lie in the order of the row's 16-byte vectors ("places": the slice's first id has place `lead`, its distance
// from the vector's start), so that rows at any alignment are read, looked up and written by whole vectors.
#include "row_types.cuh"
#include "row_team.cuh"
#include "host_error.h"
#include "launch.h"
#include <cmath>

namespace ds41 {
namespace {

constexpr int kConThreads = 512;
constexpr int kConSlice = 16384;          // ids of a CTA: 16-bit counters in 32 KB
constexpr unsigned kConListed = 0xffffu;  // counter value of an id that the bias list names (occurrences end one below)
constexpr int kConOwn = DS41_B200_CONSTRAIN_MAX_BIASES / kConThreads;  // list entries of a thread
constexpr int kConBatch = 4;              // vectors of a thread that are in flight at a time

struct ConstrainParams {
  ds41_b200_constrain_args a;
  int slice;                              // ids of a CTA, a multiple of 32
};

struct Penalty { float repetition, presence, frequency; };

// The sampler's rule, every operation rounded separately.
__device__ __forceinline__ float penalised(float x, unsigned count, const Penalty &p) {
  const float v = x > 0.f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
  return __fsub_rn(v, __fadd_rn(p.presence, __fmul_rn(p.frequency, float(count))));
}

template <class T> __device__ __forceinline__ bool fits(float y) { return finite_bits(RowType<T>::load(RowType<T>::store(y))); }

template <class T>
__global__ void __launch_bounds__(kConThreads) constrain_kernel(ConstrainParams p) {
  using R = RowType<T>;
  constexpr int kVec = R::kVec;
  __shared__ alignas(16) uint32_t counts[(kConSlice + 2 * kVec) / 2];   // 16 bits a place
  __shared__ uint32_t bits[kConSlice / 32 + 2];                          // allowed, a bit a place
  __shared__ uint32_t row_flags;                                         // 1: an allowed logit is not finite, 2: a result is not
  __shared__ int listed_twice;
  const int rank = int(team_rank()), team = int(team_size()), tid = threadIdx.x;
  const int row = int(blockIdx.x) / team;
  const int begin = min(p.a.vocab, rank * p.slice), len = min(p.a.vocab - begin, p.slice);
  for (int i = tid; i < int(sizeof(counts) / 16); i += kConThreads) reinterpret_cast<uint4 *>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) { row_flags = 0u; listed_twice = 0; }
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();

  const ds41_b200_constrain_args &a = p.a;
  const int sequence = row / a.rows_per_sequence, ahead = row - sequence * a.rows_per_sequence;
  const T *x = static_cast<const T *>(a.logits) + size_t(row) * size_t(a.logits_stride) + begin;
  T *out = static_cast<T *>(a.out) + size_t(row) * size_t(a.out_stride) + begin;
  const int lead = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % kVec);
  const bool same_places = int((reinterpret_cast<uintptr_t>(out) / sizeof(T)) % kVec) == lead;
  const T fill_value = R::store(isinf(a.fill) ? a.fill : fminf(fmaxf(a.fill, -R::kMax), R::kMax));

  // ---- the sequence's penalties and history
  Penalty pen{a.repetition, a.presence, a.frequency};
  if (a.penalties) {
    const float *own = a.penalties + size_t(sequence) * 3;
    pen = Penalty{load_input(own), load_input(own + 1), load_input(own + 2)};
  }
  int reject = 0;
  if (!(pen.repetition > 0.f) || !finite_bits(pen.repetition) || !finite_bits(pen.presence) || !finite_bits(pen.frequency))
    reject = DS41_B200_ROW_PARAMETER;
  const int drafts = a.draft_ids ? ahead : 0;
  int tokens = 0;
  if (a.history) tokens = a.history_len ? load_input(a.history_len + sequence) : int(a.history_stride);
  if (!reject && (tokens < 0 || (long long)tokens > a.history_stride || tokens > DS41_B200_CONSTRAIN_MAX_HISTORY - drafts))
    reject = DS41_B200_ROW_HISTORY;

  // ---- mask bits by place; does the mask allow any id?  (The other slices are looked at only by a CTA whose own allows none.)
  const uint32_t *mask = a.mask ? a.mask + size_t(row) * size_t(a.mask_stride) : nullptr;
  if (mask) {
    const int words = (a.vocab + 31) / 32;
    auto word = [&](int w) -> uint32_t {          // of the row, without what is behind its last id
      if (w < 0 || w >= words) return 0u;
      const uint32_t v = load_input(mask + w);
      return w == words - 1 && (a.vocab & 31) ? v & ((1u << (a.vocab & 31)) - 1u) : v;
    };
    const int first = begin / 32, own = (len + 31) / 32;
    uint32_t any = 0u;
    for (int w = tid; w <= own; w += kConThreads) {
      const uint32_t here = w < own ? word(first + w) : 0u, before = w > 0 ? word(first + w - 1) : 0u;
      any |= here;
      bits[w] = lead ? here << lead | before >> (32 - lead) : here;
    }
    if (tid == 0) bits[own + 1] = 0u;
    if (!__syncthreads_or(int(any != 0u))) {
      for (int w = tid; w < words; w += kConThreads) any |= word(w);
      if (!__syncthreads_or(int(any != 0u)) && !reject) reject = DS41_B200_ROW_EMPTY;
    }
  }
  if (reject) {                                    // the same in every CTA of the team
    const T nan = R::store(__int_as_float(0x7fffffff));
    for (int i = tid; i < len; i += kConThreads) out[i] = nan;
    if (rank == 0 && tid == 0 && a.status) a.status[row] = reject;
    return;
  }

  // ---- occurrences of this slice's ids
  __syncthreads();                                 // (the counters are zero)
  if (pen.repetition != 1.f || pen.presence != 0.f || pen.frequency != 0.f) {
    auto count = [&](int id) {
      const unsigned local = unsigned(id) - unsigned(begin);   // (padding ids, negative or beyond the vocabulary, are nobody's)
      if (local < unsigned(len)) {
        const unsigned place = local + unsigned(lead);
        atomicAdd(&counts[place >> 1], 1u << ((place & 1u) * 16u));
      }
    };
    const int32_t *h = a.history ? a.history + size_t(sequence) * size_t(a.history_stride) : nullptr;
    int i = 0;
    if ((reinterpret_cast<uintptr_t>(h) & 15u) == 0) {
      const int4 *h4 = reinterpret_cast<const int4 *>(h);
      const int vecs = tokens >> 2;
      int v = tid;
      for (; v + 7 * kConThreads < vecs; v += 8 * kConThreads) {
        int4 q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = load_input(h4 + v + k * kConThreads);
#pragma unroll
        for (int k = 0; k < 8; ++k) { count(q[k].x); count(q[k].y); count(q[k].z); count(q[k].w); }
      }
      for (; v < vecs; v += kConThreads) {
        const int4 q = load_input(h4 + v);
        count(q.x); count(q.y); count(q.z); count(q.w);
      }
      i = vecs << 2;
    }
#pragma unroll 4
    for (i += tid; i < tokens; i += kConThreads) count(load_input(h + i));
    for (int d = tid; d < drafts; d += kConThreads)
      count(load_input(a.draft_ids + size_t(sequence) * size_t(a.rows_per_sequence - 1) + d));
  }
  __syncthreads();

  auto allowed = [&](int place) { return !mask || ((bits[place >> 5] >> (place & 31)) & 1u); };
  float poison = 0.f;                              // NaN once an allowed logit is NaN or infinite
  bool over = false;

  // ---- the bias list: results of its ids from the logits as they came, before the pass over the slice (which may be in place)
  int listed[kConOwn];
  float result[kConOwn];
  if (a.biases > 0) {
    const int32_t *ids = a.bias_ids + size_t(sequence) * a.biases;
    const float *values = a.bias_values + size_t(sequence) * a.biases;
    unsigned seen[kConOwn];
#pragma unroll
    for (int k = 0; k < kConOwn; ++k) {
      const int e = tid + k * kConThreads;
      listed[k] = -1;
      if (e < a.biases) {
        const unsigned local = unsigned(load_input(ids + e)) - unsigned(begin);
        if (local < unsigned(len) && allowed(int(local) + lead)) {
          const unsigned place = local + unsigned(lead);
          listed[k] = int(local);
          result[k] = R::load(x[local]);
          seen[k] = (counts[place >> 1] >> ((place & 1u) * 16u)) & 0xffffu;
        }
      }
    }
    __syncthreads();                               // (every entry has its count)
#pragma unroll
    for (int k = 0; k < kConOwn; ++k)
      if (listed[k] >= 0) {
        const unsigned place = unsigned(listed[k] + lead), shift = (place & 1u) * 16u;
        const unsigned old = atomicOr(&counts[place >> 1], kConListed << shift);
        if (((old >> shift) & 0xffffu) == kConListed) listed_twice = 1;
      }
    __syncthreads();
    const bool twice = listed_twice != 0;
#pragma unroll
    for (int k = 0; k < kConOwn; ++k)
      if (listed[k] >= 0) {
        const int e = tid + k * kConThreads;
        float bias = load_input(values + e);
        if (twice) {                               // the id's first entry adds the later ones, which drop out
          const int id = begin + listed[k];
          bool first = true;
          for (int o = 0; o < e && first; ++o) first = load_input(ids + o) != id;
          if (!first) { listed[k] = -1; continue; }
          for (int o = e + 1; o < a.biases; ++o)
            if (load_input(ids + o) == id) bias = __fadd_rn(bias, load_input(values + o));
        }
        const float y = seen[k] ? penalised(result[k], seen[k], pen) : result[k];
        const bool was = finite_bits(result[k]);
        result[k] = __fadd_rn(y, bias);
        over |= was && !fits<T>(result[k]);
      }
  }

  // ---- the pass over the slice
  auto one = [&](T v, int place) -> T {
    if (!allowed(place)) return fill_value;
    const float f = R::load(v);
    poison = fmaf(f, 0.f, poison);
    const unsigned c = (counts[place >> 1] >> ((place & 1) * 16)) & 0xffffu;
    if (c == 0u || c == kConListed) return v;
    const float y = penalised(f, c, pen);
    over |= finite_bits(f) && !fits<T>(y);
    return R::store(y);
  };
  if (same_places) {
    const int vecs = (lead + len + kVec - 1) / kVec;
    const uint4 *x4 = reinterpret_cast<const uint4 *>(x - lead);
    uint4 *out4 = reinterpret_cast<uint4 *>(out - lead);
    constexpr unsigned kAll = (1u << kVec) - 1u;
    float fills[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) fills[i] = R::load(fill_value);
    const uint4 fill4 = R::pack(fills);
    for (int v0 = tid; v0 < vecs; v0 += kConBatch * kConThreads) {
      uint4 q[kConBatch];
      unsigned in[kConBatch];
#pragma unroll
      for (int u = 0; u < kConBatch; ++u) {
        const int v = v0 + u * kConThreads, place = v * kVec;
        in[u] = 0u;
        if (v < vecs && place >= lead && place + kVec <= lead + len) {
          in[u] = mask ? (bits[place >> 5] >> (place & 31)) & kAll : kAll;
          if (in[u]) q[u] = x4[v];
        }
      }
#pragma unroll
      for (int u = 0; u < kConBatch; ++u) {
        const int v = v0 + u * kConThreads, place = v * kVec;
        if (v >= vecs) break;
        if (place < lead || place + kVec > lead + len) {        // the slice's first or last ids
          for (int k = max(place, lead); k < min(place + kVec, lead + len); ++k) out[k - lead] = one(x[k - lead], k);
          continue;
        }
        if (!in[u]) { out4[v] = fill4; continue; }
        float y[kVec];
        R::unpack(q[u], y);
        uint32_t c[kVec / 2];
        uint32_t some = 0u;
#pragma unroll
        for (int k = 0; k < kVec / 2; ++k) { c[k] = counts[place / 2 + k]; some |= c[k]; }
#pragma unroll
        for (int k = 0; k < kVec; ++k) poison = fmaf((in[u] >> k) & 1u ? y[k] : 0.f, 0.f, poison);
        if (some) {
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            const unsigned n = (c[k / 2] >> ((k & 1) * 16)) & 0xffffu;
            if (n != 0u && n != kConListed && ((in[u] >> k) & 1u)) {
              const float z = penalised(y[k], n, pen);
              over |= finite_bits(y[k]) && !fits<T>(z);
              y[k] = z;
            }
          }
        }
        if (in[u] != kAll) {
#pragma unroll
          for (int k = 0; k < kVec; ++k) y[k] = (in[u] >> k) & 1u ? y[k] : fills[k];
        }
        out4[v] = R::pack(y);
      }
    }
  } else {                                          // rows whose vectors do not line up with the output's: id by id
#pragma unroll 4
    for (int i = tid; i < len; i += kConThreads) out[i] = one(x[i], i + lead);
  }
  if (a.biases > 0) {
    __syncthreads();                                // (the pass has written its stand-ins)
#pragma unroll
    for (int k = 0; k < kConOwn; ++k)
      if (listed[k] >= 0) out[listed[k]] = R::store(result[k]);
  }

  // ---- the row's status
  const unsigned mine = (poison == 0.f ? 0u : 1u) | (over ? 2u : 0u);
  if (__syncthreads_or(int(mine)) && mine) atomicOr(&row_flags, mine);
  team_barrier();
  if (rank == 0 && tid == 0 && a.status) {
    unsigned all = 0u;
    for (int r = 0; r < team; ++r) all |= team_read(&row_flags, r);
    a.status[row] = all & 1u ? DS41_B200_ROW_NONFINITE : all & 2u ? DS41_B200_ROW_PENALTY_OVERFLOW : 0;
  }
  team_barrier();
}

// CTAs per row: as few as the counters allow, and for batches that leave SMs idle up to eight, of at least 2048 ids each.
int constrain_team(int rows, int vocab) {
  int n = 1;
  while (n < 8 && (vocab > n * kConSlice || (2LL * rows * n <= 148 && vocab > n * 2048))) n <<= 1;
  return n;
}

template <class T>
cudaError_t launch_constrain(const ds41_b200_constrain_args &a, int rows, cudaStream_t stream) {
  const int team = constrain_team(rows, a.vocab);
  ConstrainParams p{a, ((a.vocab + team - 1) / team + 31) & ~31};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows) * unsigned(team));
  cfg.blockDim = dim3(kConThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(team); attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1] = programmatic_launch();
  cfg.attrs = attr; cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, constrain_kernel<T>, p);
}

}  // namespace
}  // namespace ds41

using namespace ds41;

extern "C" int ds41_b200_constrain_logits(const ds41_b200_constrain_args *p, cudaStream_t stream) {
  if (!p || p->struct_bytes != sizeof(ds41_b200_constrain_args)) return invalid("constrain args: struct size / ABI mismatch");
  if (p->sequences < 1 || p->rows_per_sequence < 1 || p->vocab < 1 || p->vocab > DS41_B200_MAX_VOCAB)
    return invalid("constrain args: sequences/rows/vocab out of range");
  if ((long long)p->sequences * p->rows_per_sequence > (1 << 27)) return invalid("constrain args: more than 2^27 rows");
  const int rows = p->sequences * p->rows_per_sequence;
  if (p->dtype != DS41_B200_F32 && p->dtype != DS41_B200_BF16 && p->dtype != DS41_B200_F16)
    return invalid("constrain args: rows are FP32, BF16 or FP16");
  if (!p->logits || !p->out || (p->logits_stride < p->vocab && p->logits_stride != 0) || p->out_stride < p->vocab)
    return invalid("constrain args: null buffer or short stride");
  const size_t bytes = row_type_bytes(p->dtype);
  if (reinterpret_cast<uintptr_t>(p->logits) % bytes || reinterpret_cast<uintptr_t>(p->out) % bytes)
    return invalid("constrain args: rows are not aligned to their type");
  if (!rows_apart_or_same(p->logits, p->logits_stride, p->out, p->out_stride, rows, p->vocab, bytes))
    return invalid("constrain args: out overlaps logits without being the same rows");
  if (!p->penalties && (!(p->repetition > 0) || !std::isfinite(p->repetition) || !std::isfinite(p->presence) || !std::isfinite(p->frequency)))
    return invalid("constrain args: penalties");
  if (p->history && (p->history_stride < 0 || p->history_stride > INT32_MAX ||
                     (!p->history_len && p->history_stride > DS41_B200_CONSTRAIN_MAX_HISTORY)))
    return invalid("constrain args: history longer than DS41_B200_CONSTRAIN_MAX_HISTORY");
  if (p->draft_ids && p->rows_per_sequence - 1 > DS41_B200_CONSTRAIN_MAX_HISTORY)
    return invalid("constrain args: drafts longer than DS41_B200_CONSTRAIN_MAX_HISTORY");
  if (p->biases < 0 || p->biases > DS41_B200_CONSTRAIN_MAX_BIASES || (p->biases > 0 && (!p->bias_ids || !p->bias_values)))
    return invalid("constrain args: more than DS41_B200_CONSTRAIN_MAX_BIASES biases, or no list");
  if (p->mask && p->mask_stride < (p->vocab + 31) / 32) return invalid("constrain args: mask stride shorter than the vocabulary");
  if (std::isnan(p->fill)) return invalid("constrain args: fill is NaN");
  switch (p->dtype) {
    case DS41_B200_F32: return int(launch_constrain<float>(*p, rows, stream));
    case DS41_B200_BF16: return int(launch_constrain<__nv_bfloat16>(*p, rows, stream));
    default: return int(launch_constrain<__half>(*p, rows, stream));
  }
}

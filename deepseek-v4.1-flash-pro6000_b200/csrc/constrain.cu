// Constraints on logits rows: token penalties, a bias list per sequence and the grammar bitmask, out of place or in place
// (include/ds41_b200.h has the rule).  Most of a row is only copied, or filled where the mask forbids it; few ids occur in the history
// or the bias list.  So a row is written in two steps: every 16-byte vector goes through once, allowed logits as they are, and behind a
// barrier the ids that occur or are listed are read back from the output, which holds the logit exactly, and written again.
//
// One row of 129280 fp32 ids takes 6 us (launch, the chain of loads), 48 rows with 2048 tokens 14, 256 rows with 32768 tokens, a grammar and
// biases 66, which its instructions bound: 45 M, a third of them for the histories that every CTA reads.
//
// One team of up to eight CTAs per row, each with a slice of at most 16384 ids: their occurrences fit 16-bit counters in 32 KB of
// shared memory, counted with shared-memory atomics.  Every CTA reads the whole history (from L2 after the first of them).
#include "row_types.cuh"
#include "row_team.cuh"
#include "host_error.h"
#include "launch.h"
#include <cmath>

namespace ds41 {
namespace {

constexpr int kConThreads = 512;
constexpr int kConSlice = 16384;          // ids of a CTA: 16-bit counters in 32 KB
constexpr int kConOwn = DS41_B200_CONSTRAIN_MAX_BIASES / kConThreads;  // list entries of a thread
constexpr int kConBatch = 4;              // vectors of a thread that are in flight at a time

struct ConstrainParams {
  ds41_b200_constrain_args a;
  int slice;                              // ids of a CTA, a multiple of 32
  int team;                               // CTAs of a row
};

struct Penalty { float repetition, presence, frequency; };

// The sampler's rule, every operation rounded separately.  Out of line: it is taken for few ids, from several places, and shall not
// push the loops out of the instruction cache.
__device__ __noinline__ float penalised(float x, unsigned count, Penalty p) {
  const float v = x > 0.f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
  return __fsub_rn(v, __fadd_rn(p.presence, __fmul_rn(p.frequency, float(count))));
}

template <class T, bool kTeam>
__global__ void __launch_bounds__(kConThreads, 3) constrain_kernel(ConstrainParams p) {
  using R = RowType<T>;
  constexpr int kVec = R::kVec;
  constexpr unsigned kAll = (1u << kVec) - 1u;
  __shared__ alignas(16) uint32_t counts[kConSlice / 2];   // 16 bits an id
  __shared__ uint32_t row_flags;                           // 1: an allowed logit is not finite, 2: a result is not
  __shared__ uint32_t listed_bits[kConSlice / 32];         // ids that the bias list names
  __shared__ int listed_twice;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = int(blockIdx.x) / p.team, rank = kTeam ? int(team_rank()) : int(blockIdx.x) - row * p.team;
  const int begin = min(p.a.vocab, rank * p.slice), len = min(p.a.vocab - begin, p.slice);
  for (int i = tid; i < (len + 7) / 8; i += kConThreads) reinterpret_cast<uint4 *>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
  static_assert(kConSlice == 32 * kConThreads, "32 ids a thread");
  listed_bits[tid] = 0u;
  if (tid == 0) { row_flags = 0u; listed_twice = 0; }
  __syncthreads();
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();

  const ds41_b200_constrain_args &a = p.a;
  const int sequence = a.rows_per_sequence == 1 ? row : row / a.rows_per_sequence;
  const T *x = static_cast<const T *>(a.logits) + size_t(row) * size_t(a.logits_stride) + begin;
  T *out = static_cast<T *>(a.out) + size_t(row) * size_t(a.out_stride) + begin;
  const uint32_t *mask = a.mask ? a.mask + size_t(row) * size_t(a.mask_stride) : nullptr;
  const T fill_value = R::store(isinf(a.fill) ? a.fill : fminf(fmaxf(a.fill, -R::kMax), R::kMax));

  // ---- what depends on nothing else: the thread's mask word, its entries of the bias list, its first four tokens of the history, the
  // sequence's length and penalties, all on their way at the same time
  const int lead = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % kVec);
  const bool by_vectors = int((reinterpret_cast<uintptr_t>(out) / sizeof(T)) % kVec) == lead;
  const int head = min(len, (kVec - lead) % kVec), vecs = (len - head) / kVec, tail = head + vecs * kVec;
  uint32_t word = ~0u;                             // of the 32 ids from head + 32 * tid on
  if (mask) {
    const int w = (begin >> 5) + tid, words = (a.vocab + 31) >> 5;
    word = w < words ? load_input(mask + w) : 0u;
    if (head) word = __funnelshift_r(word, w + 1 < words ? load_input(mask + w + 1) : 0u, head);
  }
  const int32_t *bias_ids = a.bias_ids + size_t(sequence) * a.biases;
  const float *bias_values = a.bias_values + size_t(sequence) * a.biases;
  int listed[kConOwn];
  float bias[kConOwn];
#pragma unroll
  for (int k = 0; k < kConOwn; ++k) {
    const int e = tid + k * kConThreads;
    listed[k] = -1; bias[k] = 0.f;
    if (e < a.biases) { listed[k] = load_input(bias_ids + e); bias[k] = load_input(bias_values + e); }
  }
  const int32_t *h = a.history ? a.history + size_t(sequence) * size_t(a.history_stride) : nullptr;
  const bool whole_vectors = (reinterpret_cast<uintptr_t>(h) & 15u) == 0;
  int4 first = make_int4(-1, -1, -1, -1);
  if (h && whole_vectors && tid < int(a.history_stride >> 2)) first = load_input(reinterpret_cast<const int4 *>(h) + tid);
  Penalty pen{a.repetition, a.presence, a.frequency};
  if (a.penalties) {
    const float *own = a.penalties + size_t(sequence) * 3;
    pen = Penalty{load_input(own), load_input(own + 1), load_input(own + 2)};
  }
  const int drafts = a.draft_ids ? row - sequence * a.rows_per_sequence : 0;
  int tokens = 0, reject = 0;
  if (h) tokens = a.history_len ? load_input(a.history_len + sequence) : int(a.history_stride);
  if (tokens < 0 || (long long)tokens > a.history_stride || tokens > DS41_B200_MAX_HISTORY - drafts) {
    reject = DS41_B200_ROW_HISTORY;
    tokens = 0;
  }

  // ---- occurrences of this slice's ids
  {
    const uint32_t base = uint32_t(__cvta_generic_to_shared(counts));
    auto count = [&](int id) {
      const unsigned local = unsigned(id) - unsigned(begin);   // (padding ids, negative or beyond the vocabulary, are nobody's)
      // a predicate, not a branch: most ids are other slices', but in nearly every warp one is this slice's
      asm volatile("{\n .reg .pred in;\n setp.lt.u32 in, %0, %1;\n @in red.shared.add.u32 [%2], %3;\n}" ::"r"(local), "r"(unsigned(len)),
                   "r"(base + ((local * 2u) & ~3u)), "r"((local & 1u) * 0xffffu + 1u) : "memory");
    };
    int i = 0;
    if (whole_vectors) {
      const int4 *h4 = reinterpret_cast<const int4 *>(h);
      const int vecs4 = tokens >> 2;
      int v = tid;
      if (v < vecs4) {
        count(first.x); count(first.y); count(first.z); count(first.w);
        v += kConThreads;
      }
      for (; v + 3 * kConThreads < vecs4; v += 4 * kConThreads) {
        int4 q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = load_input(h4 + v + k * kConThreads);
#pragma unroll
        for (int k = 0; k < 4; ++k) { count(q[k].x); count(q[k].y); count(q[k].z); count(q[k].w); }
      }
#pragma unroll 1
      for (; v < vecs4; v += kConThreads) {
        const int4 q = load_input(h4 + v);
        count(q.x); count(q.y); count(q.z); count(q.w);
      }
      i = vecs4 << 2;
    }
#pragma unroll 1
    for (i += tid; i < tokens; i += kConThreads) count(load_input(h + i));
#pragma unroll 1
    for (int d = tid; d < drafts; d += kConThreads)
      count(load_input(a.draft_ids + size_t(sequence) * size_t(a.rows_per_sequence - 1) + d));
  }

  // ---- every id once: the logit or the fill
  float poison = 0.f;                              // NaN once an allowed logit is NaN or infinite
  unsigned any = 0u;                               // an id that the mask allows
  bool over = false;
  auto allowed = [&](int local) { return !mask || ((load_input(mask + ((begin + local) >> 5)) >> ((begin + local) & 31)) & 1u); };
  auto copy = [&](int local) {
    const bool in = allowed(local);
    const T v = in ? x[local] : fill_value;
    poison = fmaf(in ? R::load(v) : 0.f, 0.f, poison);
    any |= unsigned(in);
    out[local] = v;
  };
  if (by_vectors) {
    if (tid < kVec) {                              // the ids in front of the first whole vector and behind the last
      if (tid < head) copy(tid);
    } else if (tid < 2 * kVec && tail + tid - kVec < len) {
      copy(tail + tid - kVec);
    }
    const T pair[2] = {fill_value, fill_value};
    const uint32_t f = sizeof(T) == 4 ? *reinterpret_cast<const uint32_t *>(&fill_value) : *reinterpret_cast<const uint32_t *>(pair);
    const uint4 fill4 = make_uint4(f, f, f, f);
    const int ids = min(32, max(0, vecs * kVec - 32 * tid));
    word = ids == 32 ? word : word & ((1u << ids) - 1u);
    any |= word;
    // 32 vectors a step, whose ids are those of kVec lanes' words: none of them allowed, all of them, or a mixture
    const unsigned some = __ballot_sync(0xffffffffu, word != 0u), whole = __ballot_sync(0xffffffffu, word == ~0u);
    constexpr int kSteps = 32 / kVec;
    const int v0 = warp * (1024 / kVec) + lane;
    const uint4 *x4 = reinterpret_cast<const uint4 *>(x + head) + v0;
    uint4 *out4 = reinterpret_cast<uint4 *>(out + head) + v0;
    typename R::Finite finite{};
#pragma unroll
    for (int j0 = 0; j0 < kSteps; j0 += kConBatch) {
      uint4 q[kConBatch];
#pragma unroll
      for (int u = 0; u < kConBatch; ++u) {
        q[u] = fill4;
        if (((some >> (j0 + u) * kVec) & kAll) && v0 + (j0 + u) * 32 < vecs) q[u] = x4[(j0 + u) * 32];
      }
#pragma unroll
      for (int u = 0; u < kConBatch; ++u) {
        const int j = j0 + u;
        if (((whole >> j * kVec) & kAll) == kAll) {
          finite = R::check(q[u], finite);
        } else if ((some >> j * kVec) & kAll) {
          const unsigned in = __shfl_sync(0xffffffffu, word, j * kVec + lane / kSteps) >> (lane % kSteps * kVec);
          float y[kVec];
          R::unpack(q[u], y);
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            const bool is = (in >> k) & 1u;
            poison = fmaf(is ? y[k] : 0.f, 0.f, poison);
            y[k] = is ? y[k] : R::load(fill_value);
          }
          q[u] = R::pack(y);
        }
        if (v0 + j * 32 < vecs) out4[j * 32] = q[u];
      }
    }
    if (!R::all_finite(finite)) poison = __int_as_float(0x7fffffff);
  } else {                                         // rows whose vectors do not line up with the output's: id by id
#pragma unroll 2
    for (int i = tid; i < len; i += kConThreads) copy(i);
  }
  if (!(pen.repetition > 0.f) || !finite_bits(pen.repetition) || !finite_bits(pen.presence) || !finite_bits(pen.frequency))
    reject = DS41_B200_ROW_PARAMETER;
  // (counts and copies are done.)  Does the mask allow any id?  The other slices are looked at only by a CTA whose own allows none
  if (!__syncthreads_or(int(any)) && mask) {
    const int words = (a.vocab + 31) / 32;
#pragma unroll 1
    for (int w = tid; w < words; w += kConThreads)
      any |= load_input(mask + w) & (w == words - 1 && (a.vocab & 31) ? (1u << (a.vocab & 31)) - 1u : ~0u);
    if (!__syncthreads_or(int(any)) && !reject) reject = DS41_B200_ROW_EMPTY;
  }
  if (reject) {                                    // the same in every CTA of the team
    const T nan = R::store(__int_as_float(0x7fffffff));
#pragma unroll 1
    for (int i = tid; i < len; i += kConThreads) out[i] = nan;
    if (rank == 0 && tid == 0 && a.status) a.status[row] = reject;
    return;
  }

  // ---- again the ids of the bias list, whose counters are cleared, and then those that occur
  auto settle = [&](float f, float y, int local) {
    const T v = R::store(y);
    over |= finite_bits(f) && !finite_bits(R::load(v));
    out[local] = v;
  };
  if (a.biases > 0) {
    unsigned seen[kConOwn];
#pragma unroll
    for (int k = 0; k < kConOwn; ++k) {
      const unsigned local = unsigned(listed[k]) - unsigned(begin);
      listed[k] = -1;
      if (tid + k * kConThreads < a.biases && local < unsigned(len) && allowed(int(local))) {
        listed[k] = int(local);
        seen[k] = (counts[local >> 1] >> ((local & 1u) * 16u)) & 0xffffu;
        if ((atomicOr(&listed_bits[local >> 5], 1u << (local & 31u)) >> (local & 31u)) & 1u) listed_twice = 1;
      }
    }
    __syncthreads();                               // (every entry has its count)
    const bool twice = listed_twice != 0;
#pragma unroll 1
    for (int k = 0; k < kConOwn; ++k)
      if (listed[k] >= 0) {
        atomicAnd(&counts[listed[k] >> 1], (unsigned(listed[k]) & 1u) ? 0xffffu : 0xffff0000u);   // settled here
        if (twice) {                               // the id's first entry adds the later ones, which drop out
          const int id = begin + listed[k], e = tid + k * kConThreads;
          bool is_first = true;
#pragma unroll 1
          for (int o = 0; o < e && is_first; ++o) is_first = load_input(bias_ids + o) != id;
          if (!is_first) continue;
#pragma unroll 1
          for (int o = e + 1; o < a.biases; ++o)
            if (load_input(bias_ids + o) == id) bias[k] = __fadd_rn(bias[k], load_input(bias_values + o));
        }
        const float f = R::load(out[listed[k]]);
        settle(f, __fadd_rn(seen[k] ? penalised(f, seen[k], pen) : f, bias[k]), listed[k]);
      }
  }
  if ((tokens > 0 || drafts > 0) && (pen.repetition != 1.f || pen.presence != 0.f || pen.frequency != 0.f)) {
    if (a.biases > 0) __syncthreads();
    const uint4 *quads = reinterpret_cast<const uint4 *>(counts);   // eight ids each
    const uint16_t *each = reinterpret_cast<const uint16_t *>(counts);
    uint32_t bits = 0u;                            // 16 * (id % 2) + 4 * group + id % 8 / 2
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (8 * (tid + k * kConThreads) >= len) break;
      const uint4 q = quads[tid + k * kConThreads];
      const uint32_t some = __vminu2(q.x, 0x10001u) | __vminu2(q.y, 0x10001u) << 1 | __vminu2(q.z, 0x10001u) << 2 | __vminu2(q.w, 0x10001u) << 3;
      bits |= some << (4 * k);
    }
#pragma unroll 1
    for (; bits; bits &= bits - 1u) {
      const int bit = __ffs(bits) - 1, local = 8 * (tid + ((bit >> 2) & 3) * kConThreads) + 2 * (bit & 3) + (bit >> 4);
      if (!allowed(local)) continue;
      const float f = R::load(out[local]);
      settle(f, penalised(f, each[local], pen), local);
    }
  }

  // ---- the row's status
  const unsigned mine = (poison == 0.f ? 0u : 1u) | (over ? 2u : 0u);
  if constexpr (kTeam) {
    if (__syncthreads_or(int(mine)) && mine) atomicOr(&row_flags, mine);
    team_barrier();
    if (rank == 0 && tid == 0 && a.status) {
      unsigned all = 0u;
      for (int r = 0; r < p.team; ++r) all |= team_read(&row_flags, r);
      a.status[row] = all & 1u ? DS41_B200_ROW_NONFINITE : all & 2u ? DS41_B200_ROW_PENALTY_OVERFLOW : 0;
    }
    team_barrier();
  } else {                                         // (cleared before the launch; -3 | -1 is -1)
    static_assert((DS41_B200_ROW_NONFINITE | DS41_B200_ROW_PENALTY_OVERFLOW) == DS41_B200_ROW_NONFINITE, "the first that holds");
    if (mine && a.status) atomicOr(a.status + row, mine & 1u ? DS41_B200_ROW_NONFINITE : DS41_B200_ROW_PENALTY_OVERFLOW);
  }
}

// CTAs up to which those of a row form a cluster and settle its status among themselves: as many as run at a time.  Beyond, each adds its
// flags to the status words, cleared by a node in front of the kernel, since a cluster starts when all its CTAs have a place, and
// leaves together.  Cluster / cleared words, us, fp32 rows with 2048 tokens: 129280 ids 1 row 6.0 / 8.3, 32 rows 11.7 / 14.3, 48 rows 14.2 / 16.5,
// 96 rows 27.2 / 26.7, 256 rows 68 / 55; 32000 ids 96 rows 11.6 / 14.4, 256 rows 26.9 / 26.5.
constexpr int kConTeamCtas = 3 * 148;

// CTAs per row: as few as the counters allow, and for batches that leave SMs idle up to eight, of at least 2048 ids each.  Two CTAs / up to
// eight for 32000 ids, us: 1 row 7.4 / 4.9, 24 rows 10.3 / 5.8, 32 rows 10.3 / 6.6.
int constrain_team(int rows, int vocab) {
  int n = (vocab + kConSlice - 1) / kConSlice;
  while (n < 8 && 2LL * rows * n <= 148 && vocab > n * 2048) ++n;
  return n;
}

template <class T>
cudaError_t launch_constrain(const ds41_b200_constrain_args &a, int rows, cudaStream_t stream) {
  const int team = constrain_team(rows, a.vocab);
  ConstrainParams p{a, ((a.vocab + team - 1) / team + 31) & ~31, team};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(rows) * unsigned(team));
  cfg.blockDim = dim3(kConThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0] = programmatic_launch();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(team); attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 2;
  if ((long long)rows * team <= kConTeamCtas || !a.status) return cudaLaunchKernelEx(&cfg, constrain_kernel<T, true>, p);
  cfg.numAttrs = 1;
  const cudaError_t e = cudaMemsetAsync(a.status, 0, size_t(rows) * sizeof(int32_t), stream);
  if (e != cudaSuccess) return e;
  return cudaLaunchKernelEx(&cfg, constrain_kernel<T, false>, p);
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
                     (!p->history_len && p->history_stride > DS41_B200_MAX_HISTORY)))
    return invalid("constrain args: history longer than DS41_B200_MAX_HISTORY");
  if (p->draft_ids && p->rows_per_sequence - 1 > DS41_B200_MAX_HISTORY)
    return invalid("constrain args: drafts longer than DS41_B200_MAX_HISTORY");
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

// Distillation of logits rows from a teacher's top logits: loss, gradient, or both in one call (include/ds41_b200.h has the formulas).
//
// With S_r = sum over the ids outside the list of exp((z_i - m_r) / T), m_r their maximum, the gradient of those ids is one factor per
// row times the exponential that the sum was made of,
//   g_i = T scale (q_rest - rest) exp((z_i - m_r) / T) / S_r,
// and the listed ids are few.  So the sum leaves the listed ids out (no difference of nearly equal sums where the student is sure of the
// list), the list's own terms and everything per row are taken in FP64 by few threads, and the gradient pass multiplies by one number.
//
// Here a team of up to eight CTAs takes a row, each a slice of it that stays in shared memory, so that the row is read once, and goes on to
// the next row of its own.  In a CTA, the compute warps run over the slice: a running maximum and sum per thread, one exchange of
// (maximum, sum) between all warps of the team, then the gradient from shared memory.  A thread's vectors are its own from the
// asynchronous copy on (no barrier between copy and use), and where it has written a vector's gradient it starts the copy of the
// next row's.  Two more warps: one gathers and reduces the next row's list and sets the last row's listed ids; the other brings the next
// row's mask and, a row behind, takes the loss in FP64.  Three CTAs share an SM, each at another point of its row.  Small batches are bound
// by the list's chain of loads and the exchange (8 rows of 129280 bf16 ids 8.1 us the loss, 10.5 with the gradient), masked ones by the
// instructions of the mask (450 rows of 65537 fp32 ids 114 us, 0.37 of the copy rate).  Many long rows go through distill_stream.cuh.
#include "distill_stream.cuh"
#include "row_team.cuh"
#include "host_error.h"
#include <type_traits>

namespace ds41 {
namespace {

template <int kCompute>
struct DistillSmem {
  DistillRow rows[4];                         // by the number of the row's turn: the last one, this one, the next two
  float2 sums[4][kCompute / 32];              // every warp's (maximum, sum), read by the team
  float2 result[2];                           // (maximum, sum) of the row's ids outside the list
  float2 all[2];                              // of all its ids: the maximum, 1 / the sum; a NaN where the gradient has no listed ids to set
};

// Words of bits for a slice of so many bytes.
template <int kCompute> __host__ __device__ __forceinline__ int distill_bit_words(int bytes) {
  return (bytes / 16 + 1 + kDisGroup * kCompute - 1) / (kDisGroup * kCompute) * kCompute;
}

template <class T, int kMode, int kCompute>
__global__ void __launch_bounds__(kCompute + 64, kCompute == 256 ? 3 : 8) distill_kernel(DistillParams p) {
  using R = RowType<T>;
  constexpr int kVec = R::kVec, kWarps = kCompute / 32;
  constexpr unsigned kAll = (1u << kVec) - 1u;
  extern __shared__ uint4 stage[];            // the slice, by vectors; behind it two rows' bits, weights, logits and ids of the list
  __shared__ DistillSmem<kCompute> s;
  const ds41_b200_distill_args &a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = int(team_rank()), teams = int(gridDim.x) / p.team, own_team = int(blockIdx.x) / p.team;
  const int begin = min(a.vocab, rank * p.slice), len = min(a.vocab - begin, p.slice);
  const int top_room = (a.top + 3) & ~3, bits_room = distill_bit_words<kCompute>(p.slice * int(sizeof(T)));
  uint4 *const behind = stage + p.slice * int(sizeof(T)) / 16 + 1;
  double *const weights = reinterpret_cast<double *>(behind);
  int *const ids = reinterpret_cast<int *>(weights + 2 * top_room);
  float *const zs = reinterpret_cast<float *>(ids + 2 * top_room);
  // which ids are in the sum (allowed and not listed): a word holds the bits of the four vectors that a thread takes together
  uint32_t *const bits = reinterpret_cast<uint32_t *>(zs + 2 * top_room);
  uint32_t *const mask_words = bits + 2 * bits_room;   // of the slice, as they come, and a zero
  const int mask_room = p.slice / 32 + 1;
  auto bit_word = [](int v) { return v / (kDisGroup * kCompute) * kCompute + v % kCompute; };
  auto bit_shift = [](int v) { return v / kCompute % kDisGroup * kVec; };
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();

  // the copies of a group of the thread's vectors
  auto start_copies = [&](const DistillSlice<T, kCompute> &c, int at) {
    const uint32_t to = uint32_t(__cvta_generic_to_shared(stage + tid + at));
#pragma unroll
    for (int u = 0; u < kDisGroup; ++u)
      if (c.whole(at + u * kCompute))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * kCompute * 16), "l"(c.from + at + u * kCompute) : "memory");
    if (c.any_partial()) {
#pragma unroll 1
      for (int i = at; i < min(c.mine, at + kDisGroup * kCompute); i += kCompute)
        if (!c.whole(i)) {
          const int v = tid + i;
          copy_ids<T>(reinterpret_cast<T *>(stage) + c.lead, c.x, max(0, v * kVec - c.lead), min(len, (v + 1) * kVec - c.lead));
        }
    }
    copies_commit();
  };

  // ---- the list of the row of turn `turn`, by one warp
  auto list_of = [&](int turn) { return DistillList{weights + (turn & 1) * top_room, ids + (turn & 1) * top_room, zs + (turn & 1) * top_room}; };
  auto take_list = [&](int row, int turn) {
    const DistillList list = list_of(turn);
    gather_list<T, kMode>(p, row, s.rows[turn & 3], list, lane);
    barrier_of<2, 64>();                      // (the bits are set)
    const DistillSlice<T, kCompute> c(p, row, begin, len, 0);
    uint32_t *const out = bits + (turn & 1) * bits_room;
#pragma unroll 1
    for (int e = lane; e < a.top; e += 32) {
      const unsigned local = unsigned(list.ids[e]) - unsigned(begin);
      if (local < unsigned(len)) {
        const int place = int(local) + c.lead, v = place / kVec;
        atomicAnd(&out[bit_word(v)], ~(1u << (bit_shift(v) + place % kVec)));
      }
    }
  };
  // ---- by the other: the bits of its allowed ids
  auto take_bits = [&](int row, int turn) {
    const DistillSlice<T, kCompute> c(p, row, begin, len, 0);
    uint32_t *const out = bits + (turn & 1) * bits_room;
    if (a.mask) {
      const uint32_t *from = a.mask + size_t(row) * size_t(a.mask_stride) + begin / 32;
      uint32_t *const words = mask_words + (turn & 1) * mask_room;
      const int count = min(p.slice / 32, (a.vocab + 31) / 32 - begin / 32);
#pragma unroll 4
      for (int w = lane; w < count; w += 32)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(uint32_t(__cvta_generic_to_shared(words + w))), "l"(from + w) : "memory");
      if (lane == 0) words[max(count, 0)] = 0u;
      copies_commit();
    }
    for (int w = lane; w < bits_room / 4; w += 32) reinterpret_cast<uint4 *>(out)[w] = make_uint4(~0u, ~0u, ~0u, ~0u);
    copies_wait(0);
    __syncwarp();
    if (lane == 0) {                          // nothing in front of the slice's first place or behind its last
      out[0] &= ~((1u << c.lead) - 1u);
      const int behind = c.vecs * kVec - c.lead - len, v = c.vecs - 1;
      if (behind > 0) out[bit_word(v)] &= ~(((1u << behind) - 1u) << (bit_shift(v) + kVec - behind));
    }
    barrier_of<2, 64>();
  };
  // (maximum, sum) of the ids outside the list of the turn's row, from the whole team's warps: 64 at most, in the same order everywhere
  auto combine = [&](int turn) {
    float most = -FLT_MAX, sum = 0.f;
    for (int w = lane; w < kWarps * p.team; w += 32) {
      const float2 its = team_read(&s.sums[turn & 3][w % kWarps], w / kWarps);
      const float high = fmaxf(most, its.x);
      sum = sum * exp2_approx((most - high) * p.log2e_t) + its.y * exp2_approx((its.x - high) * p.log2e_t);
      most = high;
    }
    float all = most;
#pragma unroll
    for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    sum *= exp2_approx((most - all) * p.log2e_t);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return make_float2(all, sum);
  };
  // The team's CTAs wait for one another once a row: for each other's sums, and until each has read of the row what it needs of other
  // slices.  The loss alone is not waited for by the compute warps until they have the next row's sums.
  const bool together = p.team > 1 && (kMode != kDistillGrad || p.in_place);
  const int turns = (a.rows - own_team + teams - 1) / teams;
  for (int turn = -1; turn <= turns; ++turn) {  // (one ahead for the first list and copies, one behind for the last loss)
    const int row = own_team + turn * teams, next = row + teams;
    const bool has = turn >= 0 && turn < turns, has_next = turn + 1 < turns;
    if (warp >= kWarps) {                     // a row ahead, and a row behind
      if (kMode == kDistillLoss) {
        if (together && turn > 0) team_wait();
        if (warp > kWarps && turn > 0 && rank == 0) {
          const float2 both = combine(turn - 1);
          if (lane == 0) s.result[(turn - 1) & 1] = both;
          __syncwarp();
        }
      }
      if (together && has) team_arrive();
      if (warp == kWarps) {
        if (kMode != kDistillLoss && turn > 0) set_listed<T>(p, row - teams, s.rows[(turn - 1) & 3], list_of(turn - 1), s.result[(turn - 1) & 1], s.all[(turn - 1) & 1], begin, len, lane);
        if (has_next) take_list(next, turn + 1);
      } else {
        if (lane == 0) s.rows[(turn + 2) & 3].scale = row_scale_of<kMode>(p, next + teams);
        if (lane == 0 && turn < 0) s.rows[0].scale = row_scale_of<kMode>(p, next);
        if (has_next) take_bits(next, turn + 1);
        if (kMode != kDistillGrad && rank == 0 && lane == 0 && turn > 0) finish_row<kMode>(p, row - teams, s.rows[(turn - 1) & 3], s.result[(turn - 1) & 1]);
      }
      if (kMode != kDistillLoss && together && has) team_wait();
    } else if (!has) {
      if (kMode == kDistillLoss && together && turn > 0) team_wait();
      if (has_next && row_scale_of<kMode>(p, next) != 0.f) {
        const DistillSlice<T, kCompute> c(p, next, begin, len, tid);
#pragma unroll 1
        for (int g = 0; g < kDisGroups; ++g) start_copies(c, g * kDisGroup * kCompute);
      }
    } else {
      const DistillRow &r = s.rows[turn & 3];
      const DistillSlice<T, kCompute> c(p, row, begin, len, tid), c_next(p, has_next ? next : row, begin, len, tid);
      const bool skip = skipped<kMode>(r), ahead = has_next && !skipped<kMode>(s.rows[(turn + 1) & 3]);
      const uint32_t *const in_sum = bits + (turn & 1) * bits_room + tid;
      const float log2e_t = p.log2e_t;
      T *const grad = kMode == kDistillLoss ? nullptr : static_cast<T *>(a.grad) + size_t(row) * size_t(a.grad_stride) + begin;
      const bool by_vectors = kMode != kDistillLoss && int((reinterpret_cast<uintptr_t>(grad) / sizeof(T)) % kVec) == c.lead;
      // f(at) over the thread's vectors by groups.  arrive: as their copies do; start_next: behind each group the copies of the next
      // row's, so that as many groups are on their way as before
      auto run = [&](auto arrive, auto start_next, auto f) {
#pragma unroll 1
        for (int g = 0; g < kDisGroups; ++g) {
          const int at = g * kDisGroup * kCompute;
          if (arrive.value) copies_wait(kDisGroups - 1 - (start_next.value && ahead ? 0 : g));
          if (at < c.mine) f(at);
          if (start_next.value && ahead) start_copies(c_next, at);
        }
      };
      using Yes = std::true_type;
      using No = std::false_type;
      constexpr uint32_t kNone = sizeof(T) == 4 ? 0xffff0000u : 0u;     // (a word's bits that are no vector's)
      // the thread's vectors of a group, ids that are not in the sum as -inf; keep: in the stage too
      auto take = [&](int at, bool keep, uint4 (&q)[kDisGroup]) {
        uint4 *const here = stage + tid + at;
        if (at + (kDisGroup - 1) * kCompute < c.mine) {
#pragma unroll
          for (int u = 0; u < kDisGroup; ++u) q[u] = here[u * kCompute];
        } else {
#pragma unroll
          for (int u = 0; u < kDisGroup; ++u) {
            q[u] = R::nothing();
            if (at + u * kCompute < c.mine) q[u] = here[u * kCompute];
          }
        }
        uint32_t in = in_sum[at / kDisGroup] | kNone;
        if (a.mask) {
          const uint32_t *const words = mask_words + (turn & 1) * mask_room;
#pragma unroll
          for (int u = 0; u < kDisGroup; ++u) {
            const int first = (tid + at + u * kCompute) * kVec - c.lead;   // the vector's first id in the slice
            uint32_t some = 0u;
            if (first < 0) some = words[0] << -first;
            else if (first < len) some = __funnelshift_r(words[first >> 5], words[(first >> 5) + 1], first & 31);
            in &= ~((~some & kAll) << (u * kVec));
          }
        }
        if (in != ~0u) {
#pragma unroll
          for (int u = 0; u < kDisGroup; ++u) {
            q[u] = R::only(q[u], in >> (u * kVec));
            if (keep && at + u * kCompute < c.mine) here[u * kCompute] = q[u];
          }
        }
      };

      // ---- maximum and sum of the ids outside the list
      float high = -FLT_MAX, high_c = -INFINITY, sums[4] = {0.f, 0.f, 0.f, 0.f};   // (relative to high_c)
      auto add = [&](int at) {
        uint4 q[kDisGroup];
        take(at, kMode == kDistillBoth, q);
        const float top = R::largest(q);
        if (top > high) {
          const float top_c = rounded_product(top, log2e_t);
          const float down = rise(high, high_c, top, top_c, log2e_t);
#pragma unroll
          for (int i = 0; i < 4; ++i) sums[i] *= down;
          high = top; high_c = top_c;
        }
        const bool is_near = near_exponent(high_c);
        const float scaled = is_near ? log2e_t : 1.f, minus = is_near ? -high_c : -high;
#pragma unroll
        for (int u = 0; u < kDisGroup; ++u) {
          float y[kVec];
          R::unpack(q[u], y);
          if (is_near) {
#pragma unroll
            for (int k = 0; k < kVec; ++k) sums[k % 4] += exp2_approx(fmaf(y[k], scaled, minus));
          } else {
#pragma unroll
            for (int k = 0; k < kVec; ++k) sums[k % 4] += exp2_approx(fmaf(y[k], scaled, minus) * log2e_t);
          }
        }
      };
      if (kMode == kDistillLoss) run(Yes{}, Yes{}, add);
      if (kMode == kDistillBoth && !skip) run(Yes{}, No{}, add);
      if (kMode != kDistillGrad) {
        float all = high;
#pragma unroll
        for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
        float sum = ((sums[0] + sums[1]) + (sums[2] + sums[3])) * exp2_approx(-excess(high, log2e_t, high_c));   // relative to high
        sum *= exp2_approx((high - all) * log2e_t);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s.sums[turn & 3][warp] = make_float2(all, sum);
      }
      float rest_max = -FLT_MAX, rest_sum = 0.f;
      if (kMode == kDistillLoss) {
        if (together) {
          if (turn > 0) team_wait();          // (for the row before)
          team_arrive();
        }
      } else if (together) {
        team_barrier();
      } else if (kMode == kDistillBoth) {
        barrier_of<1, kCompute>();
      }
      if (kMode == kDistillBoth) {
        const float2 both = combine(turn);
        rest_max = both.x; rest_sum = both.y;
      }

      // ---- the gradient
      if (kMode != kDistillLoss) {
        const DistillFactors f = gradient_factors<kMode, sizeof(T)>(p, r, rest_max, rest_sum);
        const bool fill = skip || f.reject != 0;
        if (tid == 0) {
          s.result[turn & 1] = make_float2(f.rest_max, f.rest_sum);
          s.all[turn & 1] = make_float2(f.largest, fill ? __int_as_float(0x7fffffff) : f.inverse_sum);
        }
        uint4 *const to = reinterpret_cast<uint4 *>(grad - c.lead) + tid;
        auto finish_vector = [&](float (&y)[kVec]) {
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < kVec; ++k) y[k] *= f.size;
          }
          uint4 g = R::pack(y);
          if constexpr (sizeof(T) != 4) g = make_uint4(g.x ^ f.sign, g.y ^ f.sign, g.z ^ f.sign, g.w ^ f.sign);
          return g;
        };
        auto step = [&](int at) {
          uint4 q[kDisGroup];
          if (kMode == kDistillGrad) {
            take(at, false, q);
          } else {
#pragma unroll
            for (int u = 0; u < kDisGroup; ++u)
              if (at + u * kCompute < c.mine) q[u] = stage[tid + at + u * kCompute];
          }
#pragma unroll
          for (int u = 0; u < kDisGroup; ++u) {
            float y[kVec];
            R::unpack(q[u], y);
            if (f.close) {
#pragma unroll
              for (int k = 0; k < kVec; ++k) y[k] = exp2_approx(fmaf(y[k], log2e_t, f.offset));
            } else {
#pragma unroll
              for (int k = 0; k < kVec; ++k) y[k] = exp2_approx(fmaf(y[k], f.scaled, f.minus) * f.factor + f.shift);
            }
            q[u] = finish_vector(y);
            if (by_vectors && c.whole(at + u * kCompute)) to[at + u * kCompute] = q[u];
          }
          if (!by_vectors || c.any_partial()) {   // by way of the stage, where the vectors are not needed any more
#pragma unroll
            for (int u = 0; u < kDisGroup; ++u)
              if (at + u * kCompute < c.mine) stage[tid + at + u * kCompute] = q[u];
#pragma unroll 1
            for (int i = at; i < min(c.mine, at + kDisGroup * kCompute); i += kCompute) {
              if (by_vectors && c.whole(i)) continue;
              const int v = tid + i;
              copy_ids<T>(grad, reinterpret_cast<const T *>(stage) + c.lead, max(0, v * kVec - c.lead), min(len, (v + 1) * kVec - c.lead));
            }
          }
        };
        if (!fill) {
          run(std::integral_constant<bool, kMode == kDistillGrad>{}, Yes{}, step);
        } else {                              // (a row that was rejected, or is padding)
          if (!skip) copies_wait(0);
          run(No{}, Yes{}, [](int) {});
          const T each = !skip && f.reject != DS41_B200_ROW_EMPTY ? R::store(__int_as_float(0x7fffffff)) : R::store(0.f);
          const T pair[2] = {each, each};
          const uint32_t w = sizeof(T) == 4 ? *reinterpret_cast<const uint32_t *>(&each) : *reinterpret_cast<const uint32_t *>(pair);
#pragma unroll 1
          for (int i = 0; i < c.mine; i += kCompute) {
            if (by_vectors && c.whole(i)) to[i] = make_uint4(w, w, w, w);
            else {
#pragma unroll 1
              for (int k = max(0, (tid + i) * kVec - c.lead); k < min(len, (tid + i + 1) * kVec - c.lead); ++k) grad[k] = each;
            }
          }
        }
      }
    }
    __syncthreads();
  }
  if (p.team > 1) team_barrier();
}

constexpr int kStreamRows = 148;
constexpr int kStreamSmem = 111 * 1024;       // two CTAs an SM

// Teams that the GPU holds at a time (asked of the runtime once per variant, device, team and shared memory of a thread's calls).
template <class T, int kMode, int kCompute>
cudaError_t resident_teams(const cudaLaunchConfig_t &cfg, int dev, int team, int *teams) {
  static thread_local struct { int dev, team, teams; size_t smem; } known{-1, 0, 0, 0};
  if (known.dev != dev) {
    const cudaError_t e = cudaFuncSetAttribute(distill_kernel<T, kMode, kCompute>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    if (e != cudaSuccess) return e;
  }
  if (known.dev != dev || known.team != team || known.smem != cfg.dynamicSmemBytes) {
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, distill_kernel<T, kMode, kCompute>, &cfg);
    if (e != cudaSuccess) return e;
    known = {dev, team, n < 1 ? 1 : n, cfg.dynamicSmemBytes};
  }
  *teams = known.teams;
  return cudaSuccess;
}

template <int kCompute> size_t distill_smem(int slice, const ds41_b200_distill_args &a, size_t bytes) {
  return size_t(slice) * bytes + 16 + 2 * size_t((a.top + 3) & ~3) * 16 + 2 * size_t(distill_bit_words<kCompute>(slice * int(bytes))) * 4 +
         (a.mask ? 2 * (size_t(slice) / 32 + 1) * 4 : 0);
}

template <class T, int kMode, int kCompute>
cudaError_t launch_distill(const DistillParams &p, cudaStream_t stream) {
  int dev = 0, teams = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(p.team));
  cfg.blockDim = dim3(kCompute + 64);
  cfg.dynamicSmemBytes = distill_smem<kCompute>(p.slice, p.a, sizeof(T));
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(p.team); attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1] = programmatic_launch();
  cfg.attrs = attr; cfg.numAttrs = 1;
  e = resident_teams<T, kMode, kCompute>(cfg, dev, p.team, &teams);
  if (e != cudaSuccess) return e;
  // as many rows for every team, if not one less
  const int turns = (p.a.rows + teams - 1) / teams;
  cfg.gridDim = dim3(unsigned((p.a.rows + turns - 1) / turns) * unsigned(p.team));
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, kMode, kCompute>, p);
}

template <class T, int kMode>
cudaError_t launch_stream(const DistillParams &p, size_t smem, cudaStream_t stream) {
  static thread_local struct { int dev, ctas; size_t smem; } known{-1, 0, 0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (known.dev != dev || known.smem != smem) {
    int per_sm = 0, sms = 0;
    e = cudaFuncSetAttribute(distill_stream_kernel<T, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamSmem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, distill_stream_kernel<T, kMode>, kStreamThreads + 64, smem);
    if (e != cudaSuccess) return e;
    known = {dev, per_sm * sms < 1 ? 1 : per_sm * sms, smem};
  }
  const int turns = (p.a.rows + known.ctas - 1) / known.ctas;
  return launch_early(distill_stream_kernel<T, kMode>, (p.a.rows + turns - 1) / turns, kStreamThreads + 64, smem, stream, p);
}

template <class T, int kMode>
cudaError_t launch_distill(DistillParams &d, cudaStream_t stream) {
  // Long rows, and enough of them for one CTA each.  Team / stream, us a call, 129280 ids: bf16 loss and gradient 100 rows 24.7 / 24.3, 148 rows
  // 36 / 26, 600 rows 93 / 90, 1024 rows 148 / 123; bf16 loss 148 rows 23 / 18, 1024 rows 84 / 61; fp32 loss 148 rows 32 / 24, 1024 rows 146 / 94;
  // the gradient alone, and fp32 loss and gradient from 600 rows on, within 6 % of each other
  d.groups = stream_groups(d.a.vocab, RowType<T>::kVec);
  const size_t smem = size_t(kStreamRing) * kDisGroup * kStreamThreads * 16 + 2 * size_t((d.a.top + 3) & ~3) * 16 + 2 * size_t(stream_marks<T>(d.groups));
  if (!d.a.mask && d.a.top < 256 && d.groups >= kStreamRing && d.a.rows >= kStreamRows && smem <= kStreamSmem) return launch_stream<T, kMode>(d, smem, stream);
  constexpr int kSmall = 64 * kDisVectors * 16 / int(sizeof(T)), kLarge = 4 * kSmall;   // ids of a CTA
  const int vocab = d.a.vocab;
  // CTAs per row: as few as hold it, three CTAs to an SM where eight of them can, and for batches that leave SMs idle up to eight, of at least
  // 4096 ids each (8 rows of 129280 bf16 ids, loss and gradient: four CTAs 12.6 us, eight 10.5)
  auto slice = [&](int team) { return ((vocab + team - 1) / team + 31) & ~31; };
  d.team = 1;
  while (d.team < 8 && (slice(d.team) > kLarge || distill_smem<256>(slice(d.team), d.a, sizeof(T)) > 74 * 1024)) ++d.team;
  while (d.team < 8 && 2LL * d.a.rows * d.team <= 148 && vocab > d.team * 4096) ++d.team;
  d.slice = slice(d.team);
  // Few compute threads a CTA where there are more rows than the wide ones take at a time.  64 / 256 threads, us, bf16 loss and gradient, one
  // CTA per row: 4000 ids 128 rows 9.6 / 8.7, 600 rows 12.1 / 17.6, 5000 rows 51 / 91; 1031 ids 600 rows 10.6 / 17.3
  return d.slice <= kSmall && (long long)d.a.rows * d.team > 3 * 148 ? launch_distill<T, kMode, 64>(d, stream) : launch_distill<T, kMode, 256>(d, stream);
}

template <int kMode>
int distill(const ds41_b200_distill_args *p, cudaStream_t stream) {
  if (!p || p->struct_bytes != sizeof(ds41_b200_distill_args)) return invalid("distill args: struct size / ABI mismatch");
  if (p->rows < 1 || p->rows > (1 << 27) || p->vocab < 1 || p->vocab > DS41_B200_MAX_VOCAB) return invalid("distill args: rows/vocab out of range");
  if (p->dtype != DS41_B200_F32 && p->dtype != DS41_B200_BF16 && p->dtype != DS41_B200_F16)
    return invalid("distill args: rows are FP32, BF16 or FP16");
  if (p->teacher_dtype != DS41_B200_F32 && p->teacher_dtype != DS41_B200_F64) return invalid("distill args: teacher values are FP32 or FP64");
  if (p->top < 1 || p->top > DS41_B200_DISTILL_MAX_TOP) return invalid("distill args: top out of range");
  if (p->reserved != 0 || (p->tail != 0 && p->tail != 1)) return invalid("distill args: tail is 0 or 1");
  if (!(p->temperature >= 1e-3 && p->temperature <= 1e3)) return invalid("distill args: temperature out of range");
  if (p->tail && p->temperature != 1.0) return invalid("distill args: the tail's log-probabilities are those of temperature 1");
  const size_t bytes = row_type_bytes(p->dtype), value_bytes = p->teacher_dtype == DS41_B200_F64 ? 8 : 4;
  if (!p->logits || p->logits_stride < p->vocab || reinterpret_cast<uintptr_t>(p->logits) % bytes)
    return invalid("distill args: logits: null, short stride or not aligned to their type");
  if (!p->teacher_ids || !p->teacher_values || p->ids_stride < p->top || p->values_stride < p->top ||
      reinterpret_cast<uintptr_t>(p->teacher_ids) % 4 || reinterpret_cast<uintptr_t>(p->teacher_values) % value_bytes)
    return invalid("distill args: teacher: null, short stride or not aligned to their type");
  if (p->mask && p->mask_stride < (p->vocab + 31) / 32) return invalid("distill args: mask stride shorter than the vocabulary");
  if (reinterpret_cast<uintptr_t>(p->stats) % 16) return invalid("distill args: stats are not 16-byte aligned");
  if (kMode != kDistillGrad && (!p->loss || !p->status)) return invalid("distill args: no loss or status buffer");
  if (kMode == kDistillGrad && !p->stats) return invalid("distill args: the gradient needs the forward pass's stats");
  if (kMode == kDistillLoss && (p->row_scale || p->grad)) return invalid("distill args: row_scale and grad belong to the gradient's calls");
  if (kMode != kDistillLoss) {
    if (!p->grad || p->grad_stride < p->vocab || reinterpret_cast<uintptr_t>(p->grad) % bytes)
      return invalid("distill args: grad: null, short stride or not aligned to its type");
    if (!rows_apart_or_same(p->logits, p->logits_stride, p->grad, p->grad_stride, p->rows, p->vocab, bytes))
      return invalid("distill args: grad overlaps logits without being the same rows");
  }
  DistillParams d{*p, p->grad == p->logits, 0, 1, 0, float(1.4426950408889634 / p->temperature), 1.0 / p->temperature};
  switch (p->dtype) {
    case DS41_B200_F32: return int(launch_distill<float, kMode>(d, stream));
    case DS41_B200_BF16: return int(launch_distill<__nv_bfloat16, kMode>(d, stream));
    default: return int(launch_distill<__half, kMode>(d, stream));
  }
}

}  // namespace
}  // namespace ds41

using namespace ds41;

extern "C" int ds41_b200_distill_loss(const ds41_b200_distill_args *args, cudaStream_t stream) { return distill<kDistillLoss>(args, stream); }
extern "C" int ds41_b200_distill_grad(const ds41_b200_distill_args *args, cudaStream_t stream) { return distill<kDistillGrad>(args, stream); }
extern "C" int ds41_b200_distill_loss_grad(const ds41_b200_distill_args *args, cudaStream_t stream) { return distill<kDistillBoth>(args, stream); }

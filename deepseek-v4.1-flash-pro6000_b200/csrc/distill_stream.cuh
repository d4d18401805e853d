// The distillation of many long rows without a mask: one CTA per row, no team.  A row does not fit a CTA's shared memory, so it is
// streamed through a ring of groups (four vectors of each thread): once for the sum, and for the gradient a second time from its end to
// its beginning, where the groups read last are still in the ring and those before them are the latest in the L2.  A group's copy
// starts when the group in its place has been used, whichever pass or row it belongs to, so that copies are always on their way; the
// list of a row, its reductions and the loss are one warp's work per row instead of one per slice.
// The loss is bound by memory (1024 rows of 129280 fp32 ids 95 us, 0.85 of the copy rate); loss and gradient by two exponentials an id
// (4096 bf16 rows 456 us, 0.71: its DRAM traffic at 0.86 of the copy rate, the exponential's pipe busy 0.53 of the time).  Two CTAs an SM: the rows of three
// do not fit the L2 until they are read again (511 us).
#pragma once
#include "distill_row.cuh"
#include <type_traits>

namespace ds41 {
namespace {

constexpr int kStreamThreads = 384;           // compute threads; two CTAs to an SM
constexpr int kStreamRing = 4;                // groups on their way or in use

struct DistillStreamSmem {
  DistillRow rows[4];                         // by the number of the row's turn: the last one, this one, the next two
  float2 sums[4][kStreamThreads / 32];
  float2 result[2], all[2];                   // as in DistillSmem
  uint8_t next[2][256];                       // of a list's entries: another one of the same thread and groups (1 up; 0: none)
};

// Entries by the thread and group (FP32: pair of groups) that hold their id.
template <class T> __host__ __device__ constexpr int stream_marks(int groups) { return (sizeof(T) == 4 ? (groups + 1) / 2 : groups) * kStreamThreads; }
inline int stream_groups(int vocab, int vec) { return (vocab + 2 * (vec - 1)) / vec / (kDisGroup * kStreamThreads) + 1; }

template <class T, int kMode>
__global__ void __launch_bounds__(kStreamThreads + 64, 2) distill_stream_kernel(DistillParams p) {
  using R = RowType<T>;
  constexpr int kVec = R::kVec, kWarps = kStreamThreads / 32, kStride = kDisGroup * kStreamThreads;
  extern __shared__ uint4 stage[];            // the ring; behind it two rows' marks, weights, logits and ids of the list
  __shared__ DistillStreamSmem s;
  const ds41_b200_distill_args &a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, groups = p.groups;
  const int top_room = (a.top + 3) & ~3, marks_room = stream_marks<T>(groups);
  double *const weights = reinterpret_cast<double *>(stage + kStreamRing * kStride);
  int *const ids = reinterpret_cast<int *>(weights + 2 * top_room);
  float *const zs = reinterpret_cast<float *>(ids + 2 * top_room);
  uint32_t *const marks = reinterpret_cast<uint32_t *>(zs + 2 * top_room);   // bytes: an entry, 1 up; 0: none
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();

  const int rows_apart = int(gridDim.x), first_row = int(blockIdx.x);
  const int turns = (a.rows - first_row + rows_apart - 1) / rows_apart;
  // Where a group lies in the ring: a single pass goes on where the row before has ended; the two passes of loss and gradient end with
  // group 0, from where the next row counts the other way
  auto place_of = [&](int turn, int g) {
    if (kMode == kDistillBoth) return (turn & 1 ? kStreamRing - 1 - g % kStreamRing : g % kStreamRing) * kStride;
    return int((unsigned(turn) * unsigned(groups) + unsigned(g)) % kStreamRing) * kStride;
  };
  // the ids of vector v that are the row's
  auto ids_from = [&](const DistillSlice<T, kStreamThreads> &c, int v) { return max(0, v * kVec - c.lead); };
  auto ids_to = [&](const DistillSlice<T, kStreamThreads> &c, int v) { return min(a.vocab, (v + 1) * kVec - c.lead); };
  // whether all vectors of a group, every thread's, are whole ones of the row
  auto inner = [&](const DistillSlice<T, kStreamThreads> &c, int g) { return (g > 0 || c.lead == 0) && (g + 1) * kStride <= (c.lead + a.vocab) / kVec; };
  // the copies of a group; what is not the row's is -inf
  auto start_group = [&](const DistillSlice<T, kStreamThreads> &c, int g, int place, bool is) {
    const int at = g * kStride;
    uint4 *const here = stage + place + tid;
    const uint32_t to = uint32_t(__cvta_generic_to_shared(here));
    if (is && inner(c, g)) {
      const uint4 *const from = c.from + at;
#pragma unroll
      for (int u = 0; u < kDisGroup; ++u)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * kStreamThreads * 16), "l"(from + u * kStreamThreads) : "memory");
    } else if (is) {
#pragma unroll
      for (int u = 0; u < kDisGroup; ++u) {
        if (c.whole(at + u * kStreamThreads))
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * kStreamThreads * 16), "l"(c.from + at + u * kStreamThreads) : "memory");
        else
          here[u * kStreamThreads] = R::nothing();
      }
      if (c.any_partial()) {
#pragma unroll 1
        for (int u = 0; u < kDisGroup && at + u * kStreamThreads < c.mine; ++u)
          if (!c.whole(at + u * kStreamThreads)) {
            const int v = tid + at + u * kStreamThreads;
            copy_ids<T>(reinterpret_cast<T *>(here + u * kStreamThreads) + c.lead - v * kVec, c.x, ids_from(c, v), ids_to(c, v));
          }
      }
    }
    copies_commit();
  };
  auto list_of = [&](int turn) { return DistillList{weights + (turn & 1) * top_room, ids + (turn & 1) * top_room, zs + (turn & 1) * top_room}; };
  auto combine = [&](int turn) {
    const float2 its = lane < kWarps ? s.sums[turn & 3][lane] : make_float2(-FLT_MAX, 0.f);
    float all = its.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    float sum = its.y * exp2_approx((its.x - all) * p.log2e_t);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return make_float2(all, sum);
  };

  for (int turn = -1; turn <= turns; ++turn) {  // (one ahead for the first list and copies, one behind for the last loss)
    const int row = first_row + turn * rows_apart, next = row + rows_apart;
    const bool has = turn >= 0 && turn < turns, has_next = turn + 1 < turns;
    if (warp == kWarps) {                     // the list of the next row, the listed ids of the last one
      if (kMode != kDistillLoss && turn > 0)
        set_listed<T>(p, row - rows_apart, s.rows[(turn - 1) & 3], list_of(turn - 1), s.result[(turn - 1) & 1], s.all[(turn - 1) & 1], 0, a.vocab, lane);
      if (has_next) {
        const DistillList list = list_of(turn + 1);
        gather_list<T, kMode>(p, next, s.rows[(turn + 1) & 3], list, lane);
        barrier_of<2, 64>();                  // (the marks are zero)
        const DistillSlice<T, kStreamThreads> c(p, next, 0, a.vocab, 0);
        uint32_t *const out = marks + ((turn + 1) & 1) * (marks_room / 4);
#pragma unroll 1
        for (int e = lane; e < a.top; e += 32) {
          if (list.ids[e] < 0) continue;
          const int v = (list.ids[e] + c.lead) / kVec, g = v / kStride;
          const int mark = (sizeof(T) == 4 ? g / 2 : g) * kStreamThreads + v % kStreamThreads, shift = mark % 4 * 8;
          uint32_t seen = out[mark / 4], was;
          do {                                // (in front of those that are there: some lane's turn ends with every round)
            was = seen;
            s.next[(turn + 1) & 1][e] = uint8_t(was >> shift);
            seen = atomicCAS(&out[mark / 4], was, (was & ~(255u << shift)) | unsigned(e + 1) << shift);
          } while (seen != was);
        }
      }
    } else if (warp > kWarps) {               // the loss of the last row
      if (lane == 0) s.rows[(turn + 2) & 3].scale = row_scale_of<kMode>(p, next + rows_apart);
      if (lane == 0 && turn < 0) s.rows[0].scale = row_scale_of<kMode>(p, next);
      if (has_next) {
        uint4 *const out = reinterpret_cast<uint4 *>(marks + ((turn + 1) & 1) * (marks_room / 4));
        for (int i = lane; i < marks_room / 16; i += 32) out[i] = make_uint4(0u, 0u, 0u, 0u);
        barrier_of<2, 64>();
      }
      if (kMode == kDistillLoss && turn > 0) {
        const float2 both = combine(turn - 1);
        if (lane == 0) s.result[(turn - 1) & 1] = both;
      }
      if (kMode != kDistillGrad && lane == 0 && turn > 0) finish_row<kMode>(p, row - rows_apart, s.rows[(turn - 1) & 3], s.result[(turn - 1) & 1]);
    } else if (!has) {
      const bool is = has_next && row_scale_of<kMode>(p, next) != 0.f;
      const DistillSlice<T, kStreamThreads> c(p, has_next ? next : first_row, 0, a.vocab, tid);
#pragma unroll 1
      for (int g = 0; g < kStreamRing; ++g) start_group(c, g, place_of(turn + 1, g), is);
    } else {
      const DistillRow &r = s.rows[turn & 3];
      const DistillSlice<T, kStreamThreads> c(p, row, 0, a.vocab, tid), c_next(p, has_next ? next : row, 0, a.vocab, tid);
      const bool skip = skipped<kMode>(r), ahead = has_next && !skipped<kMode>(s.rows[(turn + 1) & 3]);
      const uint8_t *const mark_of = reinterpret_cast<const uint8_t *>(marks + (turn & 1) * (marks_room / 4)) + tid;
      const int *const listed = list_of(turn).ids;
      const float log2e_t = p.log2e_t;
      auto mark = [&](int g) { return unsigned(mark_of[(sizeof(T) == 4 ? g / 2 : g) * kStreamThreads]); };
      // the thread's vectors of a group that has arrived, listed ids as -inf
      auto take = [&](int g, int place, uint4 (&q)[kDisGroup]) {
        uint4 *const here = stage + place + tid;
#pragma unroll 1
        for (unsigned entry = mark(g); entry; entry = s.next[turn & 1][entry - 1]) {
          const int at = listed[entry - 1] + c.lead, v = at / kVec - g * kStride - tid;
          if (unsigned(v) < unsigned(kStride)) reinterpret_cast<T *>(here + v)[at % kVec] = R::store(-INFINITY);
        }
#pragma unroll
        for (int u = 0; u < kDisGroup; ++u) q[u] = here[u * kStreamThreads];
      };

      // ---- maximum and sum of the ids outside the list, forwards
      float high = -FLT_MAX, high_c = -INFINITY, sums[4] = {0.f, 0.f, 0.f, 0.f};   // (relative to high_c)
      float rest_max = -FLT_MAX, rest_sum = 0.f;
      if (kMode != kDistillGrad && !skip) {
#pragma unroll 1
        for (int g = 0; g < groups; ++g) {
          const int place = place_of(turn, g);
          copies_wait(kStreamRing - 1);
          uint4 q[kDisGroup];
          take(g, place, q);
          const float top = R::largest(q);
          if (top > high) {
            const float top_c = rounded_product(top, log2e_t);
            const float down = rise(high, high_c, top, top_c, log2e_t);
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[i] *= down;
            high = top; high_c = top_c;
          }
          if (near_exponent(high_c)) {
#pragma unroll
            for (int u = 0; u < kDisGroup; ++u) {
              float y[kVec];
              R::unpack(q[u], y);
#pragma unroll
              for (int k = 0; k < kVec; ++k) sums[k % 4] += exp2_approx(fmaf(y[k], log2e_t, -high_c));
            }
          } else {
#pragma unroll 1
            for (int u = 0; u < kDisGroup; ++u) {
              float y[kVec];
              R::unpack(stage[place + tid + u * kStreamThreads], y);
#pragma unroll
              for (int k = 0; k < kVec; ++k) sums[k % 4] += exp2_approx((y[k] - high) * log2e_t);
            }
          }
          const int after = g + kStreamRing;  // (what the ring holds at the end of a first pass stays for the second)
          if (kMode == kDistillLoss && after >= groups) start_group(c_next, after - groups, place, ahead);
          else start_group(c, after, place, after < groups);
        }
      }
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
      if (kMode == kDistillBoth) {
        barrier_of<1, kStreamThreads>();
        const float2 both = combine(turn);
        rest_max = both.x; rest_sum = both.y;
      }

      // ---- the gradient, backwards behind a sum
      if (kMode != kDistillLoss) {
        T *const grad = static_cast<T *>(a.grad) + size_t(row) * size_t(a.grad_stride);
        const bool by_vectors = int((reinterpret_cast<uintptr_t>(grad) / sizeof(T)) % kVec) == c.lead;
        uint4 *const to = reinterpret_cast<uint4 *>(grad - c.lead) + tid;
        const DistillFactors f = gradient_factors<kMode, sizeof(T)>(p, r, rest_max, rest_sum);
        const bool fill = skip || f.reject != 0;
        if (tid == 0) {
          s.result[turn & 1] = make_float2(f.rest_max, f.rest_sum);
          s.all[turn & 1] = make_float2(f.largest, fill ? __int_as_float(0x7fffffff) : f.inverse_sum);
        }
        auto finish_vector = [&](float (&y)[kVec]) {
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < kVec; ++k) y[k] *= f.size;
          }
          uint4 q = R::pack(y);
          if constexpr (sizeof(T) != 4) q = make_uint4(q.x ^ f.sign, q.y ^ f.sign, q.z ^ f.sign, q.w ^ f.sign);
          return q;
        };
        if (!fill) {
#pragma unroll 1
          for (int i = 0; i < groups; ++i) {
            const int g = kMode == kDistillBoth ? groups - 1 - i : i, place = place_of(turn, g), at = g * kStride;
            copies_wait(kStreamRing - 1);
            uint4 q[kDisGroup];
            take(g, place, q);
            const bool straight = f.close && by_vectors && inner(c, g);
            if (f.close) {
              uint4 *const to_group = to + at;
#pragma unroll
              for (int u = 0; u < kDisGroup; ++u) {
                float y[kVec];
                R::unpack(q[u], y);
#pragma unroll
                for (int k = 0; k < kVec; ++k) y[k] = exp2_approx(fmaf(y[k], log2e_t, f.offset));
                q[u] = finish_vector(y);
                if (straight) to_group[u * kStreamThreads] = q[u];
              }
            }
            if (!straight) {                  // by way of the ring, where the vectors are not needed any more
              uint4 *const here = stage + place + tid;
              if (f.close) {
#pragma unroll
                for (int u = 0; u < kDisGroup; ++u) here[u * kStreamThreads] = q[u];
              }
#pragma unroll 1
              for (int u = 0; u < kDisGroup && at + u * kStreamThreads < c.mine; ++u) {
                if (!f.close) {
                  float y[kVec];
                  R::unpack(here[u * kStreamThreads], y);
#pragma unroll
                  for (int k = 0; k < kVec; ++k) y[k] = exp2_approx(fmaf(y[k], f.scaled, f.minus) * f.factor + f.shift);
                  here[u * kStreamThreads] = finish_vector(y);
                }
                const int v = tid + at + u * kStreamThreads;
                if (by_vectors && c.whole(at + u * kStreamThreads)) to[at + u * kStreamThreads] = here[u * kStreamThreads];
                else copy_ids<T>(grad, reinterpret_cast<const T *>(here + u * kStreamThreads) + c.lead - v * kVec, ids_from(c, v), ids_to(c, v));
              }
            }
            const int after = i + kStreamRing;
            if (after >= groups) start_group(c_next, after - groups, place, ahead);
            else start_group(c, kMode == kDistillBoth ? g - kStreamRing : after, place, true);
          }
        } else {                              // (a row that was rejected, or is padding)
          copies_wait(0);
#pragma unroll 1
          for (int g = 0; g < kStreamRing; ++g) start_group(c_next, g, place_of(turn + 1, g), ahead);
          const T each = !skip && f.reject != DS41_B200_ROW_EMPTY ? R::store(__int_as_float(0x7fffffff)) : R::store(0.f);
          const T pair[2] = {each, each};
          const uint32_t w = sizeof(T) == 4 ? *reinterpret_cast<const uint32_t *>(&each) : *reinterpret_cast<const uint32_t *>(pair);
#pragma unroll 1
          for (int i = 0; i < c.mine; i += kStreamThreads) {
            if (by_vectors && c.whole(i)) to[i] = make_uint4(w, w, w, w);
            else {
#pragma unroll 1
              for (int k = ids_from(c, tid + i); k < ids_to(c, tid + i); ++k) grad[k] = each;
            }
          }
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace ds41

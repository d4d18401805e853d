// Distillation of logits rows from a teacher's top logits: loss, gradient, or both in one call (include/ds41_b200.h has the formulas).
//
// With S_r = sum over the ids outside the list of exp((z_i - m_r) / T), m_r their maximum, the gradient of those ids is one factor per
// row times the exponential that the sum was made of,
//   g_i = T scale (q_rest - rest) exp((z_i - m_r) / T) / S_r,
// and the listed ids are few.  So the sum leaves the listed ids out (no difference of nearly equal sums where the student is sure of the
// list), the list's own terms and everything per row are taken in FP64 by few threads, and the gradient pass multiplies by one number.
//
// One team of up to eight CTAs per row, each with a slice of at most 64 KB that stays in shared memory: the row is read once, by
// asynchronous copies into which each thread's own vectors come back to it (no barrier between copy and use), while the list is
// gathered and reduced.  A running maximum and sum per thread, one exchange of (maximum, sum) between the CTAs, then the gradient from
// shared memory.  Three CTAs share an SM, so that one reads while another writes.
#include "packed_fma.cuh"
#include "row_types.cuh"
#include "row_team.cuh"
#include "host_error.h"
#include "launch.h"
#include <cfloat>
#include <cmath>

namespace ds41 {
namespace {

enum DistillMode { kDistillLoss, kDistillGrad, kDistillBoth };
constexpr int kDisBytes = 65536;              // of a CTA's slice
constexpr int kDisIds = kDisBytes / 2;
constexpr int kDisTop = DS41_B200_DISTILL_MAX_TOP;
constexpr int kDisGroups = 8;                 // copies of a thread that are waited for one by one
constexpr double kDisMost = 1.01;             // what a list's probabilities may add up to: 1, and the rounding of stored values

struct DistillParams {
  ds41_b200_distill_args a;
  int slice, team;                            // ids of a CTA (a multiple of 32), CTAs of a row
  float log2e_t;                              // log2(e) / T
};

__device__ __forceinline__ void copy16_async(const void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

__device__ __forceinline__ float exp2_approx(float x) {   // 2 ulp; 0 for -inf and below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What the list amounts to, the same in every CTA of the team.
struct ListSums {
  double named, kept, entropy, share;         // sums of w over all entries in the vocabulary and over those that count, of
};                                            // w (ln w - (z - zmax) / T), of exp((z - zmax) / T); one entry per id

template <int kThreads>
struct DistillSmem {
  uint32_t bits[kDisIds / 32 + 2];            // by place: allowed and not listed
  int4 ids[kDisTop / 4];
  double weights[kDisTop];
  ListSums list[kThreads / 32];
  float2 list_max[kThreads / 32];             // (largest value, largest logit) of the entries that count
  float2 warp_sum[kThreads / 32];             // (maximum, sum) of the ids outside the list
  float2 slot;                                // this CTA's, read by the others
  double list_scale, log_sum;                 // of the row: what follows from all of it
  double total, largest;
  float coef, rest_max;
  int reject;
};

template <class T, int kMode, int kThreads>
__global__ void __launch_bounds__(kThreads, 1536 / kThreads) distill_kernel(DistillParams p) {
  using R = RowType<T>;
  constexpr int kVec = R::kVec, kWarps = kThreads / 32, kOwn = kDisTop / kThreads > 0 ? kDisTop / kThreads : 1;
  constexpr unsigned kAll = (1u << kVec) - 1u;
  extern __shared__ uint4 stage[];            // the slice, by vectors of the row: place 0 is where its first id's vector begins
  __shared__ DistillSmem<kThreads> s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = int(blockIdx.x) / p.team, rank = int(team_rank());
  const int begin = min(p.a.vocab, rank * p.slice), len = min(p.a.vocab - begin, p.slice);
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();

  const ds41_b200_distill_args &a = p.a;
  const T *whole = static_cast<const T *>(a.logits) + size_t(row) * size_t(a.logits_stride), *x = whole + begin;
  T *grad = kMode == kDistillLoss ? nullptr : static_cast<T *>(a.grad) + size_t(row) * size_t(a.grad_stride) + begin;
  const uint32_t *mask = a.mask ? a.mask + size_t(row) * size_t(a.mask_stride) : nullptr;
  const int lead = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % kVec);
  const int vecs = (lead + len + kVec - 1) / kVec;
  const bool by_vectors = kMode != kDistillLoss && int((reinterpret_cast<uintptr_t>(grad) / sizeof(T)) % kVec) == lead;
  auto partial = [&](int v) { return v * kVec < lead || (v + 1) * kVec > lead + len; };
  // the gradient of vector v; ids outside the slice are not this CTA's
  auto put = [&](int v, const uint4 &q) {
    if (by_vectors && !partial(v)) {
      reinterpret_cast<uint4 *>(grad - lead)[v] = q;
    } else {
      const T *each = reinterpret_cast<const T *>(&q);
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const int i = v * kVec + k - lead;
        if (i >= 0 && i < len) grad[i] = each[k];
      }
    }
  };
  float scale = 1.f;
  if (kMode != kDistillLoss && a.row_scale) {
    scale = load_input(a.row_scale + row);
    if (scale == 0.f) {                       // padding: the same in every CTA of the team
      for (int v = tid; v < vecs; v += kThreads) put(v, make_uint4(0u, 0u, 0u, 0u));
      if (kMode == kDistillBoth && rank == 0 && tid == 0) {
        a.loss[row] = 0.f;
        a.status[row] = 0;
        if (a.stats) reinterpret_cast<float4 *>(a.stats)[row] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      return;
    }
  }

  // ---- the slice on its way; a vector that is not whole comes by its ids
#pragma unroll
  for (int g = 0; g < kDisGroups; ++g) {
    for (int v = tid + g * kThreads; v < vecs; v += g < kDisGroups - 1 ? vecs : kThreads) {
      if (partial(v)) {
        T *each = reinterpret_cast<T *>(&stage[v]);
        for (int k = 0; k < kVec; ++k) {
          const int i = v * kVec + k - lead;
          if (i >= 0 && i < len) each[k] = x[i];
        }
      } else {
        copy16_async(&stage[v], reinterpret_cast<const uint4 *>(x - lead) + v);
      }
    }
    copies_commit();
  }

  // ---- the list: what counts of it, and where it lies
  for (int w = tid; w <= (lead + len) / 32; w += kThreads) {
    uint32_t in = ~0u;
    if (mask) {
      const int first = begin / 32, words = (a.vocab + 31) / 32;
      auto word = [&](int at) { return at >= 0 && at < words ? load_input(mask + at) : 0u; };
      in = lead ? word(first + w) << lead | word(first + w - 1) >> (32 - lead) : word(first + w);
    }
    const int low = lead - 32 * w, high = lead + len - 32 * w;        // of the slice's places
    if (low > 0) in &= low < 32 ? ~0u << low : 0u;
    if (high < 32) in &= high > 0 ? (1u << high) - 1u : 0u;
    s.bits[w] = in;
  }
  int id[kOwn];
  float z[kOwn];
  double value[kOwn], weight[kOwn];
  bool counts[kOwn], named[kOwn], bad = false;
  float most = -FLT_MAX, zmax = -FLT_MAX;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int e = tid + k * kThreads;
    id[k] = -1; z[k] = 0.f; value[k] = 0.0; weight[k] = 0.0;
    if (e < a.top) {
      id[k] = load_input(a.teacher_ids + size_t(row) * size_t(a.ids_stride) + e);
      const size_t at = size_t(row) * size_t(a.values_stride) + e;
      value[k] = a.teacher_dtype == DS41_B200_F64 ? load_input(static_cast<const double *>(a.teacher_values) + at)
                                                  : double(load_input(static_cast<const float *>(a.teacher_values) + at));
    }
    named[k] = id[k] >= 0 && id[k] < a.vocab;
    counts[k] = named[k] && (!mask || ((load_input(mask + (id[k] >> 5)) >> (id[k] & 31)) & 1u));
    if (counts[k]) z[k] = R::load(whole[id[k]]);
    counts[k] = counts[k] && !(z[k] == -INFINITY);
    bad |= named[k] && !(value[k] < INFINITY);
    bad |= counts[k] && !(z[k] < INFINITY);
    if (counts[k]) { most = fmaxf(most, float(value[k])); zmax = fmaxf(zmax, z[k]); }
    if (e < kDisTop) reinterpret_cast<int *>(s.ids)[e] = counts[k] ? id[k] : -2 - e;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    zmax = fmaxf(zmax, __shfl_xor_sync(0xffffffffu, zmax, o));
  }
  if (lane == 0) s.list_max[warp] = make_float2(most, zmax);
  bad = __syncthreads_or(int(bad));
  for (int w = 0; w < kWarps; ++w) { most = fmaxf(most, s.list_max[w].x); zmax = fmaxf(zmax, s.list_max[w].y); }
  const double t = a.temperature;
  bool first[kOwn], again = false;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int e = tid + k * kThreads;
    first[k] = counts[k];
    if (named[k]) weight[k] = a.tail ? exp(value[k]) : exp((value[k] - double(most)) / t);
    if (counts[k]) {
      for (int j = 0; 4 * j < e; ++j) {       // an entry of the same id in front of it?
        const int4 q = s.ids[j];
        const int before = e - 4 * j;
        if (q.x == id[k] || (before > 1 && q.y == id[k]) || (before > 2 && q.z == id[k]) || (before > 3 && q.w == id[k])) first[k] = false;
      }
      again |= !first[k];
      const unsigned local = unsigned(id[k]) - unsigned(begin);
      if (local < unsigned(len)) {
        const unsigned place = local + unsigned(lead);
        atomicAnd(&s.bits[place >> 5], ~(1u << (place & 31u)));
      }
    }
    if (e < kDisTop) s.weights[e] = counts[k] ? weight[k] : 0.0;
  }
  again = __syncthreads_or(int(again));
  ListSums sums{0.0, 0.0, 0.0, 0.0};
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    sums.named += weight[k];
    if (!first[k]) continue;
    if (again) {
      const int *ids = reinterpret_cast<const int *>(s.ids);
      for (int j = tid + k * kThreads + 1; j < a.top; ++j)
        if (ids[j] == id[k]) weight[k] += s.weights[j];
    }
    const double gap = (double(z[k]) - double(zmax)) / t;
    sums.kept += weight[k];
    if (weight[k] > 0.0) sums.entropy += weight[k] * (log(weight[k]) - gap);
    sums.share += exp(gap);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sums.named += __shfl_xor_sync(0xffffffffu, sums.named, o);
    sums.kept += __shfl_xor_sync(0xffffffffu, sums.kept, o);
    sums.entropy += __shfl_xor_sync(0xffffffffu, sums.entropy, o);
    sums.share += __shfl_xor_sync(0xffffffffu, sums.share, o);
  }
  if (lane == 0) s.list[warp] = sums;

  // ---- maximum and sum of the ids outside the list; what is left out becomes -inf in shared memory
  const float2x c2 = pack_f32x2(p.log2e_t, p.log2e_t);
  float high = -FLT_MAX;
  float2x sum2 = pack_f32x2(0.f, 0.f);
  auto take = [&](int v) {
    float y[kVec];
    R::unpack(stage[v], y);
    const unsigned in = (s.bits[v * kVec >> 5] >> (v * kVec & 31)) & kAll;
    if (in != kAll) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) y[k] = (in >> k) & 1u ? y[k] : -INFINITY;
      stage[v] = R::pack(y);
    }
    if (kMode == kDistillGrad) return;
    float top = y[0];
#pragma unroll
    for (int k = 1; k < kVec; ++k) top = fmaxf(top, y[k]);
    if (top > high) {
      const float down = exp2_approx((high - top) * p.log2e_t);
      sum2 = mul_f32x2(sum2, pack_f32x2(down, down));
      high = top;
    }
    const float2x minus = pack_f32x2(-high, -high);
#pragma unroll
    for (int k = 0; k < kVec; k += 2) {
      float e0, e1;
      unpack_f32x2(mul_f32x2(add_f32x2(pack_f32x2(y[k], y[k + 1]), minus), c2), e0, e1);
      sum2 = add_f32x2(sum2, pack_f32x2(exp2_approx(e0), exp2_approx(e1)));
    }
  };
#pragma unroll
  for (int g = 0; g < kDisGroups; ++g) {
    if (g == 0) copies_wait<7>();
    if (g == 1) copies_wait<6>();
    if (g == 2) copies_wait<5>();
    if (g == 3) copies_wait<4>();
    if (g == 4) copies_wait<3>();
    if (g == 5) copies_wait<2>();
    if (g == 6) copies_wait<1>();
    if (g == 7) copies_wait<0>();
    for (int v = tid + g * kThreads; v < vecs; v += g < kDisGroups - 1 ? vecs : kThreads) take(v);
  }
  if (kMode != kDistillGrad) {
    float s0, s1, all = high;
    unpack_f32x2(sum2, s0, s1);
#pragma unroll
    for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    float sum = (s0 + s1) * exp2_approx((high - all) * p.log2e_t);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s.warp_sum[warp] = make_float2(all, sum);
    __syncthreads();
    if (warp == 0) {
      const float2 own = lane < kWarps ? s.warp_sum[lane] : make_float2(-FLT_MAX, 0.f);
      all = own.x;
#pragma unroll
      for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
      sum = own.y * exp2_approx((own.x - all) * p.log2e_t);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) s.slot = make_float2(all, sum);
    }
  }
  team_barrier();                             // every CTA has its slot, and has read of the row what it needs of other slices
  // ---- what follows for the row, by one warp of each CTA
  if (warp == 0) {
    ListSums list{0.0, 0.0, 0.0, 0.0};
    for (int w = 0; w < kWarps; ++w) {
      list.named += s.list[w].named; list.kept += s.list[w].kept;
      list.entropy += s.list[w].entropy; list.share += s.list[w].share;
    }
    float rest_max = -FLT_MAX, rest_sum = 0.f;
    double largest, log_sum, log_rest;        // (log_rest: of the sum outside the list, relative to rest_max)
    bool any;
    if (kMode == kDistillGrad) {
      const float4 kept = reinterpret_cast<const float4 *>(a.stats)[row];
      rest_sum = kept.x == kept.x ? 0.f : kept.x;   // (NaN: the forward pass has rejected the row)
      any = kept.w > -INFINITY;
      largest = kept.x; log_sum = kept.y; rest_max = any ? kept.z : 0.f; log_rest = kept.w;
    } else {
      const float2 its = lane < p.team ? team_read(&s.slot, lane) : make_float2(-FLT_MAX, 0.f);
      rest_max = its.x;
#pragma unroll
      for (int o = 4; o; o >>= 1) rest_max = fmaxf(rest_max, __shfl_xor_sync(0xffffffffu, rest_max, o));
      rest_sum = its.y * exp2_approx((its.x - rest_max) * p.log2e_t);
#pragma unroll
      for (int o = 4; o; o >>= 1) rest_sum += __shfl_xor_sync(0xffffffffu, rest_sum, o);
      any = !(rest_sum == 0.f);
      if (!any) rest_max = -FLT_MAX;
    }
    if (lane == 0) {
      if (kMode != kDistillGrad) {
        largest = any ? double(fmaxf(rest_max, zmax)) : double(zmax);
        log_rest = log(double(rest_sum));
        log_sum = log((any ? double(rest_sum) * exp((double(rest_max) - largest) / t) : 0.0) + list.share * exp((double(zmax) - largest) / t));
      }
      int reject = 0;
      if (bad) reject = DS41_B200_ROW_NONFINITE;
      else if (a.tail && list.named > kDisMost) reject = DS41_B200_ROW_NOT_NORMALIZED;
      else if (!(list.kept > 0.0)) reject = DS41_B200_ROW_EMPTY;
      else if (!(rest_sum < INFINITY)) reject = DS41_B200_ROW_NONFINITE;
      const double rest = a.tail && any ? fmax(0.0, 1.0 - list.named) : 0.0, total = list.kept + rest, tail = rest / total;
      const double log_q = any ? (double(rest_max) - largest) / t + log_rest - log_sum : 0.0;
      const double q_rest = any ? exp(log_q) : 0.0;
      s.coef = any ? float(double(scale) * t * (q_rest - tail) * exp(-log_rest)) : 0.f;
      s.rest_max = rest_max;
      s.list_scale = double(scale) * t;
      s.total = total; s.largest = largest; s.log_sum = log_sum;
      s.reject = reject;
      if (kMode != kDistillGrad && rank == 0) {
        const double kept = list.kept / total;
        double loss = list.entropy / total - kept * log(total) - kept * ((double(zmax) - largest) / t - log_sum);
        if (tail > 0.0) loss += tail * (log(tail) - log_q);
        const float nan = __int_as_float(0x7fffffff);
        a.loss[row] = reject == 0 ? float(t * t * loss) : reject == DS41_B200_ROW_EMPTY ? 0.f : nan;
        a.status[row] = reject;
        if (a.stats)
          reinterpret_cast<float4 *>(a.stats)[row] = reject ? make_float4(nan, nan, nan, nan)
            : make_float4(float(largest), float(log_sum), any ? rest_max : -INFINITY, any ? float(log_rest) : -INFINITY);
      }
    }
  }
  team_arrive();                              // (the slots have been read)
  if (kMode != kDistillLoss) {
    __syncthreads();
    const int reject = s.reject;
    if (reject) {
      const T nan = R::store(__int_as_float(0x7fffffff));
      T each[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) each[k] = nan;
      const uint4 q = reject == DS41_B200_ROW_EMPTY ? make_uint4(0u, 0u, 0u, 0u) : *reinterpret_cast<const uint4 *>(each);
      for (int v = tid; v < vecs; v += kThreads) put(v, q);
    } else {
      const float2x minus = pack_f32x2(-s.rest_max, -s.rest_max), coef2 = pack_f32x2(s.coef, s.coef);
      for (int v = tid; v < vecs; v += kThreads) {
        float y[kVec];
        R::unpack(stage[v], y);
#pragma unroll
        for (int k = 0; k < kVec; k += 2) {
          float e0, e1;
          unpack_f32x2(mul_f32x2(add_f32x2(pack_f32x2(y[k], y[k + 1]), minus), c2), e0, e1);
          unpack_f32x2(mul_f32x2(pack_f32x2(exp2_approx(e0), exp2_approx(e1)), coef2), y[k], y[k + 1]);
        }
        put(v, R::pack(y));
      }
      __syncthreads();                        // (zeros stand where listed ids are)
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const unsigned local = unsigned(id[k]) - unsigned(begin);
        if (first[k] && local < unsigned(len)) {
          const double q = exp((double(z[k]) - s.largest) / t - s.log_sum);
          grad[local] = R::store(float(s.list_scale * (q - weight[k] / s.total)));
        }
      }
    }
  }
  team_wait();
}

template <class T, int kMode, int kThreads>
cudaError_t launch_distill(const DistillParams &p, cudaStream_t stream) {
  static thread_local int configured_device = -1;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (configured_device != dev) {
    e = cudaFuncSetAttribute(distill_kernel<T, kMode, kThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, kDisBytes + 16);
    if (e != cudaSuccess) return e;
    configured_device = dev;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(p.a.rows) * unsigned(p.team));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = size_t(p.slice) * sizeof(T) + 16;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(p.team); attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1] = programmatic_launch();
  cfg.attrs = attr; cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, distill_kernel<T, kMode, kThreads>, p);
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
  DistillParams d{*p, 0, 1, float(1.4426950408889634 / p->temperature)};
  // CTAs per row: as few as hold it, and for batches that leave SMs idle up to eight, of at least 4096 ids each
  const long long most = kDisBytes / bytes;
  d.team = int((p->vocab + most - 1) / most);
  while (d.team < 8 && 2LL * p->rows * d.team <= 148 && p->vocab > d.team * 4096) ++d.team;
  d.slice = ((p->vocab + d.team - 1) / d.team + 31) & ~31;
  switch (p->dtype) {
    case DS41_B200_F32: return int(launch_distill<float, kMode, 512>(d, stream));
    case DS41_B200_BF16: return int(launch_distill<__nv_bfloat16, kMode, 512>(d, stream));
    default: return int(launch_distill<__half, kMode, 512>(d, stream));
  }
}

}  // namespace
}  // namespace ds41

using namespace ds41;

extern "C" int ds41_b200_distill_loss(const ds41_b200_distill_args *args, cudaStream_t stream) { return distill<kDistillLoss>(args, stream); }
extern "C" int ds41_b200_distill_grad(const ds41_b200_distill_args *args, cudaStream_t stream) { return distill<kDistillGrad>(args, stream); }
extern "C" int ds41_b200_distill_loss_grad(const ds41_b200_distill_args *args, cudaStream_t stream) { return distill<kDistillBoth>(args, stream); }
